"""The operators of batched serving, as calls that can be measured: the write of
rotated keys and values into a paged KV cache, the attention of one new token
over that cache, the attention of whole (packed) prompts, and the draw of the
next token from the logits.

Each case computes in two ways: ``own = False`` in elementary torch
operations, ``own = True`` through polarflash_b200.  Sizes are this
repository's: 32 query and 8 KV heads of 128 (or 64 query heads over 8), the
small models' heads of 64, the vocabulary of 128256, and generic ones.
"""
import math
import os
import random
import sys

import torch

own = False

MODES = ("fp16", "bf16", "int8", "2bit", "2bit_asym")
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ROPE_THETA = 500000.0


def _api():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "polar-flash_b200")
    if not os.path.isdir(root):
        root = os.path.join(os.getcwd(), "polar-flash_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import polarflash_b200

    return polarflash_b200


# ---- cases -----------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 conversations: every one appends one token
        {"name": "rope_kv_decode_64_bf16", "op": "rope_kv", "seqs": 64, "new": 0, "lo": 100, "hi": 2048, "nh": 32,
         "nkv": 8, "hd": 128, "mode": "bf16", "page": 64, "emit": "fp32"},
        # eight fresh prompts enter an int8 cache, with 16-bit copies for the prompt attention
        {"name": "rope_kv_prompt_8_int8", "op": "rope_kv", "seqs": 8, "new": 1, "lo": 311, "hi": 2048, "nh": 32,
         "nkv": 8, "hd": 128, "mode": "int8", "page": 32, "emit": "bf16"},
        # one conversation at a 2048-token context: latency
        {"name": "paged_1x2048_int8", "op": "paged", "seqs": 1, "lo": 2048, "hi": 2048, "nh": 32, "nkv": 8, "hd": 128,
         "mode": "int8", "page": 64, "q": "fp32"},
        # a small model's heads, short ragged contexts, small pages
        {"name": "paged_24x900_fp16_hd64", "op": "paged", "seqs": 24, "lo": 1, "hi": 900, "nh": 4, "nkv": 2, "hd": 64,
         "mode": "fp16", "page": 16, "q": "fp16"},
        # an ordinary serving batch on a 16-bit cache
        {"name": "paged_64x4096_bf16", "op": "paged", "seqs": 64, "lo": 300, "hi": 4096, "nh": 32, "nkv": 8, "hd": 128,
         "mode": "bf16", "page": 64, "q": "bf16"},
        # few long contexts on the smallest cache, eight query heads per KV head
        {"name": "paged_8x32768_2bit_asym", "op": "paged", "seqs": 8, "lo": 9001, "hi": 32768, "nh": 64, "nkv": 8,
         "hd": 128, "mode": "2bit_asym", "page": 128, "q": "fp32"},
        # one prompt of odd length: latency
        {"name": "prompt_1x611_bf16", "op": "prompt", "seqs": 1, "lo": 611, "hi": 611, "prefix": 0, "nh": 32, "nkv": 8,
         "hd": 128, "dtype": "bf16"},
        # packed ragged prompts of a small-headed model, continuing cached prefixes
        {"name": "prompt_12x1500_fp16_hd64", "op": "prompt", "seqs": 12, "lo": 37, "hi": 1500, "prefix": 500, "nh": 16,
         "nkv": 4, "hd": 64, "dtype": "fp16"},
        # one long prompt
        {"name": "prompt_1x8192_bf16", "op": "prompt", "seqs": 1, "lo": 8192, "hi": 8192, "prefix": 0, "nh": 32,
         "nkv": 8, "hd": 128, "dtype": "bf16"},
        # the next token of one conversation, every filter on: latency
        {"name": "sample_1x128256_fp32", "op": "sample", "rows": 1, "vocab": 128256, "dtype": "fp32", "filters": "all"},
        # a serving batch, nucleus sampling only
        {"name": "sample_64x128256_fp32", "op": "sample", "rows": 64, "vocab": 128256, "dtype": "fp32",
         "filters": "top_p"},
        # a large batch of 16-bit logits (many equal values) whose rows ask for different things, greedy among them
        {"name": "sample_256x32001_bf16", "op": "sample", "rows": 256, "vocab": 32001, "dtype": "bf16",
         "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope_kv", "paged", "prompt", "sample"))
    if op == "sample":
        vocab = _log(rng, 300, 151000)
        return {"op": op, "rows": max(1, min(_log(rng, 1, 300), 8000000 // vocab)), "vocab": vocab,
                "dtype": rng.choice(("fp32", "bf16", "fp16")), "filters": rng.choice(("all", "top_p", "top_k", "mixed", "none"))}
    nkv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 7, 8))
    if op == "prompt":
        seqs = _log(rng, 1, 16)
        hi = min(_log(rng, 1, 6000), 12000 // seqs)
        hd = rng.choice((64, 128, 96, 40))
        return {"op": op, "seqs": seqs, "lo": rng.randint(1, max(1, hi)), "hi": max(1, hi),
                "prefix": rng.choice((0, 0, rng.randint(1, 800))), "nh": nkv * group if nkv * group <= 32 else 32, "nkv": nkv,
                "hd": hd, "dtype": rng.choice(("bf16", "fp16"))}
    mode, page, hd = rng.choice(MODES), rng.choice((16, 32, 64, 128)), rng.choice((64, 128))
    if op == "paged":
        seqs = _log(rng, 1, 128)
        hi = max(1, min(_log(rng, 1, 32768), 200000 // seqs))
        return {"op": op, "seqs": seqs, "lo": rng.randint(0, hi), "hi": hi, "nh": nkv * group, "nkv": nkv, "hd": hd,
                "mode": mode, "page": page, "q": rng.choice(("fp32", "fp16", "bf16"))}
    seqs, fresh = _log(rng, 1, 96), rng.randint(0, 1)
    hi = max(1, min(_log(rng, 1, 3000), 16000 // seqs))
    return {"op": op, "seqs": seqs, "new": fresh, "lo": rng.randint(1, hi), "hi": hi, "nh": nkv * group, "nkv": nkv, "hd": hd,
            "mode": mode, "page": page, "emit": rng.choice(("fp32", "fp16", "bf16"))}


def _lengths(case):
    """The sequences' lengths: spread between lo and hi (over the logarithm), hi among them."""
    lo, hi, n = case["lo"], case["hi"], case["seqs"]
    a, got = max(1, lo), []
    for i in range(n):
        f = (0.6180339887 * i) % 1.0
        got.append(int(round(math.exp(math.log(hi) * (1 - f) + math.log(a) * f))) if a < hi else hi)
    if lo == 0 and n > 1:
        got[n // 2] = 0
    return got


# ---- what a program has in hand --------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _row_bytes(mode, hd):
    return hd if mode == "int8" else hd // 4


def _quantize(x, mode):
    """Rows of x [..., hd] (fp32) as (codes, scales [...], zeros [...] or None), the compressed cache's formulas."""
    if mode in ("fp16", "bf16"):
        return x.to(DTYPES[mode]), None, None
    if mode == "int8":
        s = (x.abs().amax(-1) / 127.0).clamp_min(1e-8)
        return torch.round(x / s[..., None]).clamp(-128, 127).to(torch.int8), s, None
    if mode == "2bit":
        s, z = (x.abs().amax(-1) / 1.75).clamp_min(1e-8), None
        c = torch.floor(x / s[..., None] + 2.0)
    else:
        z = x.amin(-1)
        s = ((x.amax(-1) - z) / 3.0).clamp_min(1e-8)
        c = torch.round((x - z[..., None]) / s[..., None])
    c = c.clamp(0, 3).to(torch.uint8).unflatten(-1, (-1, 4))
    return c[..., 0] << 6 | c[..., 1] << 4 | c[..., 2] << 2 | c[..., 3], s, z


def _values(codes, s, z, mode):
    """The fp32 values that codes stand for."""
    if mode in ("fp16", "bf16"):
        return codes.float()
    if mode == "int8":
        return codes.float() * s[..., None]
    c = torch.stack((codes >> 6, codes >> 4 & 3, codes >> 2 & 3, codes & 3), -1).flatten(-2).float()
    return (c - 1.5) * s[..., None] if mode == "2bit" else c * s[..., None] + z[..., None]


def _pages(case, lens, g, fill):
    """A pool [pages, nkv, page, row] for K and for V, and a table of pages in random order (-1 behind a sequence's last)."""
    nkv, hd, page, mode = case["nkv"], case["hd"], case["page"], case["mode"]
    need = [-(-n // page) for n in lens]
    n_pages, width = sum(need) + 3, max(1, max(need))
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"table": table}
    for name in ("k", "v"):
        shape = (n_pages, nkv, page)
        if fill:
            x = torch.randn(shape + (hd,), generator=g, device="cuda")
            if name == "k":  # keys have a few large channels
                x *= 1.0 + 3.0 * (torch.rand(nkv, 1, hd, generator=g, device="cuda") > 0.95)
            c, sc, z = _quantize(x, mode)
            del x
        elif mode in ("fp16", "bf16"):
            c, sc, z = torch.zeros(shape + (hd,), dtype=DTYPES[mode], device="cuda"), None, None
        else:
            c = torch.zeros(shape + (_row_bytes(mode, hd),), dtype=torch.int8 if mode == "int8" else torch.uint8, device="cuda")
            sc = torch.zeros(shape, device="cuda")
            z = torch.zeros(shape, device="cuda") if mode == "2bit_asym" else None
        s[name], s[name + "_scales"], s[name + "_zeros"] = c, sc, z
    return s


def _starts(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "sample":
        n, vocab, f = case["rows"], case["vocab"], case["filters"]
        u = lambda: torch.rand(n, generator=g, device="cuda")  # noqa: E731
        # a few likely tokens over a broad floor, as a model's logits are
        s["logits"] = (2.0 * rand(n, vocab) + 4.0 * (torch.rand(n, vocab, generator=g, device="cuda") > 0.999)).to(DTYPES[case["dtype"]])
        s["u"] = u()
        on = lambda name: f in ("all", "mixed", name)  # noqa: E731
        s["temperature"] = 0.3 + 1.2 * u()
        s["top_k"] = (1 + 100 * u() ** 2).to(torch.int32) if on("top_k") else torch.zeros(n, dtype=torch.int32, device="cuda")
        s["top_p"] = 0.5 + 0.5 * u() if on("top_p") else torch.ones(n, device="cuda")
        s["min_p"] = 0.1 * u() if on("min_p") else torch.zeros(n, device="cuda")
        if f == "mixed":
            s["temperature"] *= u() > 0.2       # greedy rows
            s["top_k"] *= u() > 0.5
            s["top_p"] = torch.where(u() > 0.5, s["top_p"], 1.0)
            s["min_p"] *= u() > 0.5
        return s
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    lens = _lengths(case)
    if case["op"] == "prompt":
        past = [(7919 * i) % (case["prefix"] + 1) for i in range(len(lens))]
        s["cu_q"], s["cu_k"] = _starts(lens), _starts([a + b for a, b in zip(lens, past)])
        s["max_q"], s["max_k"] = max(lens), max(a + b for a, b in zip(lens, past))
        dt = DTYPES[case["dtype"]]
        s["q"] = (1.5 * rand(sum(lens), nh, hd)).to(dt)
        s["k"], s["v"] = (rand(sum(lens) + sum(past), nkv, hd).to(dt) for _ in range(2))
        return s
    s |= _pages(case, lens, g, fill=case["op"] == "paged")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["op"] == "paged":
        s["q"] = (1.5 * rand(len(lens), nh, hd)).to(DTYPES[case["q"]])
        return s
    new = lens if case["new"] else [1] * len(lens)
    s["cu"] = _starts(new)
    s["q"], s["k_new"], s["v_new"] = rand(sum(new), nh, hd), rand(sum(new), nkv, hd), rand(sum(new), nkv, hd)
    pos = torch.cat([torch.arange(a - b, a, dtype=torch.float64) for a, b in zip(lens, new)]).cuda()
    freq = ROPE_THETA ** (-torch.arange(hd // 2, dtype=torch.float64, device="cuda") / (hd // 2))
    s["cos"], s["sin"] = (pos[:, None] * freq).cos().float(), (pos[:, None] * freq).sin().float()
    return s


# ---- the plain forms -------------------------------------------------------
def _rotate(x, cos, sin):
    x1, x2 = x.chunk(2, -1)
    return torch.cat((x1 * cos - x2 * sin, x1 * sin + x2 * cos), -1)


def _plain_rope_kv(s):
    case = s["case"]
    mode, page, emit = case["mode"], case["page"], DTYPES[case["emit"]]
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    q, k, v = _rotate(s["q"], cos, sin), _rotate(s["k_new"], cos, sin), s["v_new"]
    cu = s["cu"].long()
    t = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = s["lens"].long()[seq] - (cu[seq + 1] - t)
    at, row = s["table"].long()[seq, pos // page], pos % page
    for name, x in (("k", k), ("v", v)):
        for part, y in zip(("", "_scales", "_zeros"), _quantize(x, mode)):
            if y is not None:
                s[name + part][at, :, row] = y
    return [q.to(emit)] + ([k.to(emit), v.to(emit)] if case["new"] else [])


def _plain_paged(s):
    case, q, lens = s["case"], s["q"], s["lens"].long()
    nkv, hd = case["nkv"], case["hd"]
    table = s["table"].long().clamp_min(0)
    part = lambda n: _values(s[n][table], *(None if s[n + e] is None else s[n + e][table] for e in ("_scales", "_zeros")), case["mode"])  # noqa: E731
    k, v = (part(n).transpose(1, 2).flatten(2, 3) for n in ("k", "v"))  # [seqs, nkv, width * page, hd]
    seen = torch.arange(k.shape[2], device=q.device) < lens[:, None]
    v = torch.where(seen[:, None, :, None], v, 0.0)
    score = (q.float().unflatten(1, (nkv, -1)) @ k.transpose(2, 3)) / math.sqrt(hd)
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    return (torch.where(total > 0, e / total, 0.0) @ v).flatten(1, 2).to(q.dtype)


def _plain_prompt(s):
    case, q, cq, ck = s["case"], s["q"], s["cu_q"].long(), s["cu_k"].long()
    nkv, hd = case["nkv"], case["hd"]
    at = lambda cu, n: (cu[:-1, None] + torch.arange(n, device=q.device), torch.arange(n, device=q.device) < cu.diff()[:, None])  # noqa: E731
    (iq, sq), (ik, sk) = at(cq, s["max_q"]), at(ck, s["max_k"])
    part = lambda x, i, m: torch.where(m[..., None, None], x[i.clamp_max(x.shape[0] - 1)].float(), 0.0).transpose(1, 2)  # noqa: E731
    qp, kp, vp = part(q, iq, sq).unflatten(1, (nkv, -1)), part(s["k"], ik, sk)[:, :, None], part(s["v"], ik, sk)[:, :, None]
    score = (qp / math.sqrt(hd)) @ kp.transpose(3, 4)  # [seqs, nkv, group, max_q, max_k]
    reach = torch.arange(s["max_q"], device=q.device) + (ck.diff() - cq.diff())[:, None]
    seen = torch.arange(s["max_k"], device=q.device) <= reach[:, :, None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score @ vp) / torch.where(total > 0, total, 1.0)
    return out.flatten(1, 2).transpose(1, 2)[sq].to(q.dtype)


def _plain_sample(s):
    """The draw in 64 bits: sums over the vocabulary, and values next to a border."""
    x, t = s["logits"].double(), s["temperature"].double()[:, None]
    n, vocab = x.shape
    x = torch.where(x.isnan(), -math.inf, x)
    order = torch.sort(x, dim=1, descending=True, stable=True)
    top = order.values[:, :1]
    w = torch.exp(torch.where(order.values == top, 0.0, (order.values - top) / torch.where(t > 0, t, 1.0)))
    rank = torch.arange(vocab, device=x.device)
    k = s["top_k"].long()[:, None]
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    before = torch.cat((torch.zeros(n, 1, dtype=w.dtype, device=w.device), w.cumsum(1)[:, :-1]), 1)
    p = s["top_p"].double()[:, None]
    keep = (rank == 0) | (p >= 1) | (before < p * w.sum(1, keepdim=True))
    keep &= w >= s["min_p"].double()[:, None].clamp_max(1.0)
    keep &= (t > 0) | (rank == 0)
    w = torch.zeros_like(x).scatter_(1, order.indices, torch.where(keep, w, 0.0))
    c = w.cumsum(1)
    token = (c <= s["u"].double()[:, None] * c[:, -1:]).sum(1)
    last = vocab - 1 - (w.flip(1) > 0).to(torch.int8).argmax(1)
    return torch.where(top[:, 0] > -math.inf, torch.minimum(token, last), -1)


def _own(s):
    case, P = s["case"], _api()
    if case["op"] == "sample":
        return P.sample_logits(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if case["op"] == "prompt":
        return P.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
    pages = P.KVPages(case["mode"], s["k"], s["v"], s["k_scales"], s["v_scales"], s["k_zeros"], s["v_zeros"])
    if case["op"] == "paged":
        return P.paged_attention(s["q"], pages, s["table"], s["lens"])
    q, k, v = P.paged_rope_kv(s["q"], s["k_new"], s["v_new"], s["cos"], s["sin"], pages, s["table"], s["lens"], s["cu"],
                              out_dtype=DTYPES[case["emit"]], return_kv=bool(case["new"]))
    return [q, k, v] if case["new"] else [q]


def run(s):
    if own:
        out = _own(s)
    elif s["case"]["op"] == "rope_kv":
        out = _plain_rope_kv(s)
    elif s["case"]["op"] == "paged":
        out = _plain_paged(s)
    elif s["case"]["op"] == "prompt":
        out = _plain_prompt(s)
    else:
        out = _plain_sample(s)
    if s["case"]["op"] != "rope_kv":
        return out
    # the cache is an output too: as it is held in 16 bits, else as the values that its codes stand for
    mode = s["case"]["mode"]
    held = [s[n] if mode in ("fp16", "bf16") else _values(s[n], s[n + "_scales"], s[n + "_zeros"], mode) for n in ("k", "v")]
    return {"new": out, "cache": held}


# ---- what a pass cannot do without -----------------------------------------
def work(case):
    size = {"fp32": 4, "fp16": 2, "bf16": 2}
    if case["op"] == "sample":  # one read of the logits; an exponential (taken as 10) and a sum for each
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["dtype"]] + case["rows"] * 28, "flops": 12 * n}
    lens, nh, nkv, hd = _lengths(case), case["nh"], case["nkv"], case["hd"]
    if case["op"] == "prompt":  # causal: a query at place i of n over m keys sees m - n + i + 1
        past = [(7919 * i) % (case["prefix"] + 1) for i in range(len(lens))]
        pairs = sum(n * (2 * p + n + 1) // 2 for n, p in zip(lens, past))
        return {"bytes": 2 * hd * (2 * nh * sum(lens) + 2 * nkv * (sum(lens) + sum(past))), "flops": 4 * hd * nh * pairs}
    mode = case["mode"]
    row = 2 * hd if mode in ("fp16", "bf16") else _row_bytes(mode, hd) + (8 if mode == "2bit_asym" else 4)
    if case["op"] == "paged":
        return {"bytes": 2 * sum(lens) * nkv * row + 2 * case["seqs"] * nh * hd * size[case["q"]], "flops": 4 * sum(lens) * nh * hd}
    t = sum(lens) if case["new"] else case["seqs"]
    e = size[case["emit"]]
    return {"bytes": t * (nh * hd * (4 + e) + 2 * nkv * (4 * hd + row + (e * hd if case["new"] else 0)) + 4 * hd),
            "flops": t * 3 * hd * (nh + nkv)}


# ---- the definitions in 64 bits --------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return None  # token numbers: whole values
    hd, nkv = case["hd"], case["nkv"]
    group = case["nh"] // nkv
    if case["op"] == "rope_kv":
        cos, sin = s["cos"].double()[:, None], s["sin"].double()[:, None]

        def turn(x):
            z = torch.complex(x[..., : hd // 2].double(), x[..., hd // 2:].double()) * torch.complex(cos, sin)
            return torch.cat((z.real, z.imag), -1)

        q, k, v = turn(s["q"]), turn(s["k_new"]), s["v_new"].double()
        held = [None, None]  # a code at a border between two steps has no value in 64 bits
        if case["mode"] in ("fp16", "bf16"):
            held = [s["k"].double(), s["v"].double()]
            for b, (end, a, z) in enumerate(zip(s["lens"].tolist(), s["cu"][:-1].tolist(), s["cu"][1:].tolist())):
                p = torch.arange(end - (z - a), end, device=q.device)
                page = s["table"][b].long()[p // case["page"]]
                for h, x in zip(held, (k, v)):
                    h[page, :, p % case["page"]] = x[a:z]
        return {"new": [q, k, v] if case["new"] else [q], "cache": held}
    lens = _lengths(case)
    if case["op"] == "paged":
        if sum(lens) * case["nh"] * hd > 1.6e10:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            if n == 0:
                continue
            page = s["table"][b, : -(-n // case["page"])].long()
            rows = []
            for name in ("k", "v"):
                c, sc, z = (None if s[name + e] is None else s[name + e][page].transpose(0, 1).flatten(1, 2)[:, :n] for e in ("", "_scales", "_zeros"))
                if case["mode"].startswith("2bit"):
                    c = torch.stack([c.long() // 4 ** (3 - i) % 4 for i in range(4)], -1).flatten(2)
                x = c.double() - (1.5 if case["mode"] == "2bit" else 0.0)
                x = x if sc is None else x * sc.double()[..., None]
                rows.append(x if z is None else x + z.double()[..., None])
            a = torch.einsum("hgd,htd->hgt", s["q"][b].double().view(nkv, group, hd), rows[0]) * hd ** -0.5
            out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(a, -1), rows[1]).reshape(-1, hd)
        return out
    if sum(n * n for n in lens) * case["nh"] * hd > 6e11:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b, n in enumerate(lens):
        m = ck[b + 1] - ck[b]
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(case["nh"]):
            a = s["q"][cq[b]:cq[b + 1], h].double() @ s["k"][ck[b]:ck[b + 1], h // group].double().T * hd ** -0.5
            a.masked_fill_(hidden, -math.inf)
            out[cq[b]:cq[b + 1], h] = torch.softmax(a, -1) @ s["v"][ck[b]:ck[b + 1], h // group].double()
    return out


if __name__ == "__main__":
    r = random.Random(0)
    for c in listed() + [draw(r) for _ in range(6)]:
        print(c.get("name", "drawn"), c, work(c))
