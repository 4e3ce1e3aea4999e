"""Operators of serving whose speed is watched: a cache of keys and values in 8 bits (rows written, read back and attended to), copies of
its pages, and tokens drawn with given random numbers.

The cache. Pages of `bs` tokens hold e4m3 numbers, [layers, pages, heads, bs, 128], and one scale for each page and head, a power of two: the
smallest for which the page's largest finite number is at most 448 scales. A row at offset 0 of a page begins it anew; any other row may raise
the page's scale, and then the numbers that the page holds are rounded to the new one. Infinities become the largest number of their page.

Attention of single tokens: o = sum_j p_j v_j over the tokens j < ctx of a sequence, p = softmax(scale q . k_j); zero where ctx is 0.

Drawing. w_i = exp((x_i - max x) / T), in descending order with ties to the lowest index: the first top_k of them, of these the fewest that
hold top_p of their sum, of these the ones of at least min_p; then the first index, in ascending order, at which the running sum of what is
kept exceeds u times its sum. T <= 0 takes the largest. The token's log-probability is that of T = 1 over all tokens.
"""
from __future__ import annotations

import math

import torch

own = False                      # set by whoever measures: the framework's operators, or their plain forms

HD = 128
LOWEST, HIGHEST = -120, 120      # exponents of a page's scale
_T = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------------------
def rows(seqs, tokens, start, heads, groups, bs=16, dtype="bfloat16", pad=0, **more):
    """`seqs` sequences that have `start` tokens in the cache (the last: fewer) bring up to `tokens` more; `pad` rows belong to none."""
    return {**more, "kind": "rows", "seqs": seqs, "tokens": tokens, "start": start, "heads": heads, "groups": groups, "bs": bs, "dtype": dtype,
            "pad": pad}


def attend(seqs, ctx, spread, heads, groups, bs=16, dtype="bfloat16", reach=0, **more):
    """`seqs` single tokens with contexts of up to `ctx` tokens, the shortest about `spread` percent shorter; `reach`: the longest context that
    the program allows (0: the longest that is there)."""
    return {**more, "kind": "attend", "seqs": seqs, "ctx": ctx, "spread": spread, "heads": heads, "groups": groups, "bs": bs, "dtype": dtype,
            "reach": reach}


def prefix(seqs, ctx, spread, heads, groups, bs=16, dtype="bfloat16", **more):
    """Cached rows of `seqs` sequences laid out in front of their next portions."""
    return {**more, "kind": "prefix", "seqs": seqs, "ctx": ctx, "spread": spread, "heads": heads, "groups": groups, "bs": bs, "dtype": dtype}


def fork(pairs, layers, kv, bs=16, **more):
    """`pairs` pages copied in all layers."""
    return {**more, "kind": "fork", "pairs": pairs, "layers": layers, "kv": kv, "bs": bs}


def sample(seqs, vocab, top_k, top_p, min_p, dtype="bfloat16", greedy=0, sharp=2.5, **more):
    """`seqs` rows of `vocab` logits; every `greedy`-th row (0: none) takes the largest. `sharp`: their spread."""
    return {**more, "kind": "sample", "seqs": seqs, "vocab": vocab, "top_k": top_k, "top_p": top_p, "min_p": min_p, "dtype": dtype,
            "greedy": greedy, "sharp": sharp}


def listed():
    return [
        # a decode step of one user of a Llama-2-7B shaped model: latency
        rows(1, 1, 700, 32, 1, name="rows one user"),
        # the rows of a step of prompts, two of them going on inside a page
        rows(4, 2048, 70, 32, 4, name="rows prompts"),
        # one user, a short conversation
        attend(1, 700, 0, 32, 1, name="attend one user"),
        # a full batch of chats with grouped heads, fp16, in a program that allows 4096 tokens
        attend(64, 1000, 60, 16, 4, dtype="float16", reach=4096, name="attend batch 64"),
        # few users of a Llama-2-70B shaped model with long documents
        attend(4, 30011, 30, 64, 8, name="attend long documents"),
        # the largest batch, every head with its own keys and values
        attend(128, 2048, 50, 32, 1, name="attend batch 128"),
        # a portion of one prompt of ordinary length
        prefix(1, 511, 0, 16, 4, dtype="float16", name="prefix one portion"),
        # portions of long prompts
        prefix(4, 16000, 40, 64, 8, name="prefix long prompts"),
        # the last page of a prompt that a second answer starts from
        fork(1, 32, 32, name="fork one answer"),
        # many answers at once
        fork(192, 32, 32, name="fork many answers"),
        # one user, the settings of a chat
        sample(1, 32000, 50, 0.9, 0.05, name="sample one user"),
        # a full batch over a large vocabulary, nothing cut for a part of it
        sample(256, 128000, 0, 0.95, 0.0, greedy=8, name="sample batch 256"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "rows", "attend", "attend", "attend", "prefix", "fork", "sample", "sample"])
    dt, bs = rng.choice(["bfloat16", "bfloat16", "float16"]), rng.choice([8, 16, 16, 16, 32])
    groups = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    kv = max(1, _log(rng, 1, 32) // groups)
    if kind == "rows":
        tokens = rng.choice([1, 1, _log(rng, 2, 2000)])
        seqs = _log(rng, 1, 256) if tokens == 1 else _log(rng, 1, max(1, min(64, 8000 // tokens)))
        return rows(seqs, tokens, rng.randrange(0, 300), kv * groups, groups, bs, dt, rng.choice([0, 0, 3]))
    if kind == "attend":
        seqs = _log(rng, 1, 200)
        ctx = _log(rng, 1, max(2, min(100000, 5_000_000 // (seqs * kv))))
        return attend(seqs, ctx, rng.choice([0, 30, 80, 100]), kv * groups, groups, bs, dt, rng.choice([0, 0, ctx * 2]))
    if kind == "prefix":
        seqs = _log(rng, 1, 16)
        return prefix(seqs, _log(rng, 1, max(2, min(40000, 1_000_000 // (seqs * kv)))), rng.choice([0, 50, 100]), kv * groups, groups, bs, dt)
    if kind == "fork":
        layers = rng.randrange(1, 41)
        return fork(_log(rng, 1, max(1, min(900, 100_000 // (layers * kv)))), layers, kv, bs)
    vocab = _log(rng, 300, 131000)
    return sample(_log(rng, 1, max(1, min(512, 30_000_000 // vocab))), vocab, rng.choice([0, 0, 1, 20, 50, 1000]),
                  rng.choice([1.0, 1.0, 0.9, 0.95, 0.5]), rng.choice([0.0, 0.0, 0.02, 0.1]), rng.choice(["bfloat16", "float16", "float32"]),
                  rng.choice([0, 0, 4]), rng.choice([0.5, 2.5, 5.0]))


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
def _share(i):
    """A number in [0, 1) for the i-th sequence, 0 for the first."""
    return (i * 2654435761 % 4294967296) / 4294967296


def _lengths(case):
    """Contexts of the sequences: the first has the longest; with a spread of 100 some are (nearly) empty."""
    return [int(case["ctx"] * (1 - case["spread"] / 100 * _share(i))) for i in range(case["seqs"])]


def _portions(case):
    """(tokens in the cache, tokens that come) of every sequence."""
    return [(int(case["start"] * (1 - _share(2 * i + 1) / 2)), max(1, int(case["tokens"] * (1 - 0.4 * _share(i))))) for i in range(case["seqs"])]


def _pages(shape, gen, dev):
    """Pages as they are after some use: e4m3 numbers with their scales. Some channels of a head are larger than others."""
    q = torch.empty(shape, dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty(shape[:-2], dtype=torch.float32, device=dev)
    flat, fs = q.view(-1, *shape[-2:]), scale.view(-1)
    channel = 1 + 4 * (torch.rand(HD, generator=gen, device=dev) < 0.03)
    step = max(1, (1 << 25) // (shape[-2] * HD))
    for a in range(0, flat.shape[0], step):
        n = min(step, flat.shape[0] - a)
        x = torch.randn((n, shape[-2], HD), generator=gen, device=dev) * channel
        x *= torch.exp(0.5 * torch.randn((n, 1, 1), generator=gen, device=dev))
        m, e = torch.frexp(x.abs().amax((1, 2)))
        fs[a:a + n] = torch.ldexp(torch.ones_like(m), e - 9 + (m > 0.875).int())
        flat[a:a + n] = (x / fs[a:a + n, None, None]).to(torch.float8_e4m3fn)
    return q, scale


def _tables(counts, gen, dev, spare=3):
    """Block tables of sequences with `counts` pages, from a shuffled pool: (int32 [seqs, most], pages of the pool)."""
    total = sum(counts) + spare
    perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    t = torch.zeros((len(counts), max(max(counts), 1)), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(counts):
        t[i, :n] = perm[at:at + n]
        at += n
    return t, total


def _slots(table, lo, hi, bs):
    j = torch.arange(lo, hi, device=table.device)
    return table[j // bs].long() * bs + j % bs


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    c, kind = case, case["kind"]
    s = {"kind": kind}
    if kind == "sample":
        B, V = c["seqs"], c["vocab"]
        x = torch.randn((B, V), generator=gen, device=dev) * c["sharp"]
        s["logits"] = x.to(_T[c["dtype"]])
        s["u"] = torch.rand(B, generator=gen, device=dev, dtype=torch.float64)
        t = 0.5 + torch.rand(B, generator=gen, device=dev)
        if c["greedy"]:
            t[::c["greedy"]] = 0
        s["t"] = t
        s["top_k"] = torch.full((B,), c["top_k"], dtype=torch.int32, device=dev)
        s["top_p"] = torch.full((B,), c["top_p"], dtype=torch.float32, device=dev)
        s["min_p"] = torch.full((B,), c["min_p"], dtype=torch.float32, device=dev)
        return s
    bs = c["bs"]
    if kind == "fork":
        n = 2 * c["pairs"] + 5
        s["k"], s["k_scale"] = _pages((c["layers"], n, c["kv"], bs, HD), gen, dev)
        s["v"], s["v_scale"] = _pages((c["layers"], n, c["kv"], bs, HD), gen, dev)
        order = torch.randperm(n, generator=gen, device=dev).tolist()
        s["src"], s["dst"] = order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]
        return s
    H, KV, dt = c["heads"], c["heads"] // c["groups"], _T[c["dtype"]]
    s.update(H=H, KV=KV, dtype=dt)
    width = (H + 2 * KV) * HD
    if kind == "rows":
        portions = _portions(c)
        tables, n = _tables([-(-(a + m) // bs) for a, m in portions], gen, dev)
        T = sum(m for _, m in portions) + c["pad"]
        s["x"] = torch.randn((T, width), generator=gen, device=dev).to(dt)
        s["out"] = torch.empty_like(s["x"])
        none = torch.full((c["pad"],), -1, dtype=torch.int64, device=dev)
        s["slots"] = torch.cat([_slots(tables[i], a, a + m, bs) for i, (a, m) in enumerate(portions)] + [none])
        s["pos"] = torch.cat([torch.arange(a, a + m, device=dev) for a, m in portions] + [none * 0]).to(torch.int32)
        far = max(a + m for a, m in portions)
        ang = torch.arange(far, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, HD, 2, device=dev, dtype=torch.float64) / HD)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    else:
        lens = _lengths(c)
        tables, n = _tables([-(-m // bs) for m in lens], gen, dev)
    s["k"], s["k_scale"] = _pages((n, KV, bs, HD), gen, dev)
    s["v"], s["v_scale"] = _pages((n, KV, bs, HD), gen, dev)
    if kind == "attend":
        s["q"] = torch.randn((c["seqs"], width), generator=gen, device=dev).to(dt)
        s["tables"], s["ctx"] = tables, torch.tensor(lens, dtype=torch.int32, device=dev)
        s["reach"] = c["reach"] or max(max(lens), 1)
    if kind == "prefix":
        # each sequence's cached rows, then 16 rows of its portion
        s["slots"] = torch.cat([_slots(tables[i], 0, m, bs) for i, m in enumerate(lens)])
        s["at"] = torch.cat([torch.arange(m, device=dev) + sum(lens[:i]) + 16 * i for i, m in enumerate(lens)])
        s["ext"] = torch.zeros((sum(lens) + 16 * len(lens), width), dtype=dt, device=dev)
    return s


def work(case):
    c, kind = case, case["kind"]
    if kind == "sample":
        return {"bytes": c["seqs"] * c["vocab"] * (4 if c["dtype"] == "float32" else 2) + 40 * c["seqs"], "flops": 2 * c["seqs"] * c["vocab"]}
    if kind == "fork":
        return {"bytes": 2 * c["pairs"] * c["layers"] * 2 * c["kv"] * (c["bs"] * HD + 4), "flops": 0}
    H, KV, bs = c["heads"], c["heads"] // c["groups"], c["bs"]
    if kind == "rows":
        T = sum(m for _, m in _portions(c))
        pages = sum(-(-(a + m) // bs) - a // bs for a, m in _portions(c))
        return {"bytes": (T + c["pad"]) * ((H + 2 * KV) * HD * 4 + 12) + T * 2 * KV * HD + pages * 2 * KV * 4 + min(T, max(m for _, m in _portions(c))) * HD * 4,
                "flops": 3 * T * (H + KV) * HD}
    lens = _lengths(c)
    read = sum(lens) * 2 * KV * HD + sum(-(-m // bs) for m in lens) * (8 * KV + 4)
    if kind == "prefix":
        return {"bytes": read + sum(lens) * (2 * KV * HD * 2 + 16), "flops": 2 * sum(lens) * KV * HD}
    return {"bytes": read + c["seqs"] * (2 * H * HD * 2 + 4), "flops": 4 * sum(lens) * H * HD}


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def _turn(x, pos, cos, sin, n):
    """The first n heads of the rows x rotated by their positions, rotate-half; the tables are rounded to the rows' type."""
    T = x.shape[0]
    v = x[:, :n * HD].view(T, n, 2, HD // 2).float()
    c, t = cos[pos.long()].to(x.dtype).float()[:, None], sin[pos.long()].to(x.dtype).float()[:, None]
    a, b = v[:, :, 0], v[:, :, 1]
    return torch.stack([a * c - b * t, b * c + a * t], 2).reshape(T, n * HD).to(x.dtype)


def _scale_for(largest):
    m, e = torch.frexp(largest)
    e = torch.where(largest > 0, e - 9 + (m > 0.875).int(), LOWEST).clamp(LOWEST, HIGHEST)
    return torch.ldexp(torch.ones_like(largest), e)


def _write(x, page, off, q, scale):
    """Rows x [n, heads, HD] into the pages q with their scales, at (page, off)."""
    finite = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    pages, which = torch.unique(page, return_inverse=True)
    largest = torch.zeros((len(pages), x.shape[1]), device=x.device).scatter_reduce_(0, which[:, None].expand_as(finite), finite, "amax")
    fresh = torch.zeros(len(pages), dtype=torch.bool, device=x.device)
    fresh[which[off == 0]] = True
    old = torch.where(fresh[:, None], 2.0 ** LOWEST, scale[pages])
    new = torch.maximum(old, _scale_for(largest))
    held = q[pages].float()
    q[pages] = torch.where(fresh[:, None, None, None], held, held * (old / new)[:, :, None, None]).to(torch.float8_e4m3fn)
    scale[pages] = new
    q[page, :, off] = (x / new[which][:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)


def _rows(s):
    H, KV, x = s["H"], s["KV"], s["x"]
    T, bs = x.shape[0], s["k"].shape[2]
    out = s["out"]
    out[:, :(H + KV) * HD] = _turn(x, s["pos"], s["cos"], s["sin"], H + KV)
    out[:, (H + KV) * HD:] = x[:, (H + KV) * HD:]
    ok = s["slots"] >= 0
    page, off = s["slots"][ok] // bs, s["slots"][ok] % bs
    kv = out[ok][:, H * HD:].view(-1, 2, KV, HD).float()
    _write(kv[:, 0], page, off, s["k"], s["k_scale"])
    _write(kv[:, 1], page, off, s["v"], s["v_scale"])
    return {"rows": out, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _laid_out(q, scale, tables):
    """Cached numbers of every sequence [seqs, heads, tokens, HD] in 32 bits."""
    t = tables.long()
    return (q[t].float() * scale[t][..., None, None]).transpose(1, 2).flatten(2, 3)


def _attend(s):
    H, KV, B = s["H"], s["KV"], s["q"].shape[0]
    q = s["q"][:, :H * HD].float().view(B, KV, H // KV, HD)
    k, v = _laid_out(s["k"], s["k_scale"], s["tables"]), _laid_out(s["v"], s["v_scale"], s["tables"])
    z = q @ k.transpose(2, 3) / math.sqrt(HD)
    there = (torch.arange(k.shape[2], device=z.device) < s["ctx"][:, None])[:, None, None]
    z = z.masked_fill(~there, float("-inf"))
    m = z.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(z - m)
    v = v.masked_fill(~there[:, :, 0, :, None], 0.0)
    o = p @ v / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(B, H * HD).to(s["dtype"])


def _prefix(s):
    H, KV, bs, ext = s["H"], s["KV"], s["k"].shape[2], s["ext"]
    page, off = s["slots"] // bs, s["slots"] % bs
    ext[s["at"], H * HD:(H + KV) * HD] = (s["k"][page, :, off].float() * s["k_scale"][page][..., None]).flatten(1).to(ext.dtype)
    ext[s["at"], (H + KV) * HD:] = (s["v"][page, :, off].float() * s["v_scale"][page][..., None]).flatten(1).to(ext.dtype)
    return ext


def _fork(s):
    src, dst = (torch.tensor(s[n], device=s["k"].device) for n in ("src", "dst"))
    parts = {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}
    for t in parts.values():
        t[:, dst] = t[:, src]
    return parts


def _sample(s):
    x = s["logits"].double()
    B, V = x.shape
    top, first = x.max(-1, keepdim=True)
    t = s["t"].double()[:, None]
    w = torch.exp((x - top) / torch.where(t > 0, t, 1.0))
    down, order = torch.sort(s["logits"].float(), descending=True, stable=True)
    d = w.gather(-1, order)
    rank = torch.arange(V, device=x.device)
    k = s["top_k"].long()[:, None]
    keep = (rank < torch.where(k > 0, k, V)).expand(B, V)
    run = torch.cumsum(d * keep, -1)
    p = s["top_p"].double()[:, None]
    keep = keep & ((p >= 1) | (rank <= (run < p * run[:, -1:]).sum(-1, keepdim=True)))
    keep = keep & (d >= s["min_p"].double()[:, None])
    kept = torch.zeros_like(w).scatter_(-1, order, d * keep)
    run = torch.cumsum(kept, -1)
    token = ((run > s["u"][:, None] * run[:, -1:]) & (kept > 0)).long().argmax(-1)
    token = torch.where(t[:, 0] > 0, token, first[:, 0])
    total = torch.exp(x - top).sum(-1)
    return {"token": token, "logprob": (x.gather(-1, token[:, None])[:, 0] - top[:, 0] - total.log()).float()}


def run(s):
    kind = s["kind"]
    if own:
        from dlti_b200.ops import kv8, pages, serving
        if kind == "rows":
            kv8.rope_cache8_(s["x"], s["pos"], s["cos"], s["sin"], s["slots"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["H"], s["KV"], HD,
                             out=s["out"])
            return {"rows": s["out"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if kind == "attend":
            return kv8.paged_decode8(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["tables"], s["ctx"], s["H"], s["KV"], HD,
                                     max_ctx=s["reach"])
        if kind == "prefix":
            return kv8.gather_rows8_(s["ext"], s["at"], s["slots"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["H"], s["KV"], HD)
        if kind == "fork":
            pages.copy_pages([s["k"], s["v"], s["k_scale"], s["v_scale"]], s["src"], s["dst"], page_dim=1)
            return {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}
        token, logprob = serving.sample_given(s["logits"], s["u"], s["t"], s["top_k"], s["top_p"], s["min_p"], want_logprob=True)
        return {"token": token, "logprob": logprob}
    return {"rows": _rows, "attend": _attend, "prefix": _prefix, "fork": _fork, "sample": _sample}[kind](s)


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------------------
def _e4m3(x):
    """x (float64) rounded to the nearest number of four significant bits, not finer than 2^-9, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_pages(new, page, off, q, scale):
    q, scale = q.double(), scale.double()
    for p in torch.unique(page).tolist():
        mine = page == p
        x, at = new[mine], off[mine]
        largest = x.abs().amax((0, 2))
        e = torch.ceil(torch.log2(largest.clamp_min(1e-300) / 448))
        e = torch.where(largest > 448 * torch.exp2(e), e + 1, torch.where(largest <= 448 * torch.exp2(e - 1), e - 1, e)).clamp_min(LOWEST)
        if bool((at == 0).any()):
            s = torch.exp2(e)
        else:
            s = torch.maximum(torch.exp2(e), scale[p])
            q[p] = _e4m3(q[p] * (scale[p] / s)[:, None, None])
        scale[p] = s
        q[p, :, at] = _e4m3(x / s[None, :, None]).transpose(0, 1)
    return q, scale


def _exact_token(x, u, t, top_k, top_p, min_p):
    x = x.double()
    if t <= 0:
        return int((x == x.max()).nonzero()[0])
    w = torch.softmax(x / t, -1)
    best = torch.argsort(x, descending=True, stable=True)[:top_k or len(x)]
    if top_p < 1:
        best = best[:int((w[best].cumsum(-1) < top_p * w[best].sum()).sum()) + 1]
    best = best[w[best] >= min_p * w.max()].sort().values
    run = w[best].cumsum(-1)
    return int(best[min(int((run <= u * run[-1]).sum()), len(best) - 1)])


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "fork":
        out = {}
        for n in ("k", "v", "k_scale", "v_scale"):
            t = s[n].double()
            for a, b in zip(s["src"], s["dst"]):
                t[:, b] = s[n][:, a].double()
            out[n] = t
        return out
    if kind == "sample":
        probs = torch.log_softmax(s["logits"].double(), -1)
        drawn = [_exact_token(x, *(s[n][b].item() for n in ("u", "t", "top_k", "top_p", "min_p"))) for b, x in enumerate(s["logits"])]
        return {"token": None, "logprob": probs.gather(-1, torch.tensor(drawn, device=probs.device)[:, None])[:, 0]}
    H, KV, bs = s["H"], s["KV"], s["k"].shape[2]
    if kind == "rows":
        x = s["x"].double().view(len(s["pos"]), -1, HD)
        z = torch.complex(s["cos"].to(s["dtype"]).double(), s["sin"].to(s["dtype"]).double())[s["pos"].long()][:, None]
        turned = torch.complex(x[:, :H + KV, :HD // 2].contiguous(), x[:, :H + KV, HD // 2:].contiguous()) * z
        turned = torch.cat([torch.cat([turned.real, turned.imag], -1), x[:, H + KV:]], 1)
        ok = s["slots"] >= 0
        held = turned[ok].to(s["dtype"]).double()                    # the cache takes the rows as they leave, in their type
        if len(torch.unique(s["slots"][ok] // bs)) > 3000:
            return None
        k, ks = _exact_pages(held[:, H:H + KV], s["slots"][ok] // bs, s["slots"][ok] % bs, s["k"], s["k_scale"])
        v, vs = _exact_pages(held[:, H + KV:], s["slots"][ok] // bs, s["slots"][ok] % bs, s["v"], s["v_scale"])
        return {"rows": turned.flatten(1), "k": k, "v": v, "k_scale": ks, "v_scale": vs}
    if kind == "prefix":
        out = s["ext"].double()
        for r, t in zip((s["k"], s["v"]), range(2)):
            scale = (s["k_scale"], s["v_scale"])[t]
            for h in range(KV):
                a = (H + t * KV + h) * HD
                out[s["at"], a:a + HD] = r[:, h].reshape(-1, HD)[s["slots"]].double() * scale[:, h].repeat_interleave(bs)[s["slots"]][:, None].double()
        return out
    out = torch.zeros((len(s["ctx"]), H, HD), dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["ctx"].tolist()):
        if n:
            t = s["tables"][b, :-(-n // bs)].long()
            k = (s["k"][t].double() * s["k_scale"][t].double()[:, :, None, None]).permute(1, 0, 2, 3).reshape(KV, -1, HD)[:, :n]
            v = (s["v"][t].double() * s["v_scale"][t].double()[:, :, None, None]).permute(1, 0, 2, 3).reshape(KV, -1, HD)[:, :n]
            q = s["q"][b, :H * HD].double().view(KV, H // KV, HD)
            out[b] = (torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / HD ** 0.5, -1) @ v).reshape(H, HD)
    return out.flatten(1)
