"""The 8-bit cache and the drawing of tokens in double precision, one function per rule; shares no code with the framework."""
import math

import torch

LOWEST, HIGHEST = -120, 120


def e4m3(x):
    """x (float64) rounded to four significant bits, not finer than 2^-9, ties to even; beyond 448: 448. NaN stays."""
    y = x.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def scale_of(largest: float) -> float:
    e = LOWEST
    while e < HIGHEST and largest > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotate(x, pos, cos, sin, n, hd):
    """The first n heads of the rows x (float64) by the tables' rows pos, already rounded to the rows' type."""
    y = x.clone()
    for h in range(n):
        a, b = x[:, h * hd:h * hd + hd // 2], x[:, h * hd + hd // 2:(h + 1) * hd]
        c, s = cos[pos], sin[pos]
        y[:, h * hd:h * hd + hd // 2] = a * c - b * s
        y[:, h * hd + hd // 2:(h + 1) * hd] = b * c + a * s
    return y


def write(x, slots, q, scale):
    """Rows x [n, heads, hd] (float64) into q [pages, heads, bs, hd] with scale [pages, heads] (float64, changed in place), page by page."""
    bs = q.shape[2]
    slots = slots.tolist()
    for page in sorted({s // bs for s in slots if s >= 0}):
        rows = [i for i, s in enumerate(slots) if s >= 0 and s // bs == page]
        fresh = any(slots[i] % bs == 0 for i in rows)
        for h in range(q.shape[1]):
            new = x[rows, h]
            fin = new[torch.isfinite(new)].abs()
            s = scale_of(float(fin.max()) if fin.numel() else 0.0)
            if not fresh:
                s = max(s, float(scale[page, h]))
                if s > float(scale[page, h]):
                    q[page, h] = e4m3(q[page, h] * (float(scale[page, h]) / s))
            scale[page, h] = s
            for i in rows:
                q[page, h, slots[i] % bs] = e4m3(x[i, h] / s)


def attend(q, k8, v8, ks, vs, table, ctx, H, KV, hd, scale):
    """(outputs [B, H hd], sum_j p_j |v_j|, largest sum_d |q_d k_jd| scale of every head [B, H]) in float64."""
    B, bs = q.shape[0], k8.shape[2]
    out, mag, reach = torch.zeros(B, H, hd, dtype=torch.float64), torch.zeros(B, H, hd, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        n = min(int(ctx[b]), table.shape[1] * bs)
        if n <= 0:
            continue
        pages = table[b, :-(-n // bs)].long()
        for h in range(H):
            g = h // (H // KV)
            k = (k8[pages, g].double() * ks[pages, g].double()[:, None, None]).reshape(-1, hd)[:n]
            v = (v8[pages, g].double() * vs[pages, g].double()[:, None, None]).reshape(-1, hd)[:n]
            x = q[b, h * hd:(h + 1) * hd].double()
            p = torch.softmax(k @ x * scale, 0)
            out[b, h], mag[b, h] = p @ v, p @ v.abs()
            reach[b, h] = (k.abs() @ x.abs()).max() * abs(scale)
    return out.flatten(1), mag.flatten(1), reach


def attend_error(out, mag, reach, ctx, dtype, hd):
    """How far a result may be off. One rounding to the type: half a step. Before it, a score is 128 products summed in fp32 (an addition loses at
    most 2^-22 of the running sum's bound, sum |q k|) and two products: 132 * 2^-22 of sum |q k| scale, for the token and the maximum (or the sum of
    all weights) both; a weight's own errors (exponential 2^-21, two 16-bit terms 2^-21) and one addition per 16 tokens, joins included, at 2^-22."""
    n = torch.as_tensor(ctx).double().clamp_min(0)[:, None]
    rel = 2 * 132 * 2.0 ** -22 * reach + 2.0 ** -19 + (n / 16 + 80) * 2.0 ** -22
    return torch.finfo(dtype).eps / 2 * out.abs() + (1 + torch.finfo(dtype).eps) * mag * rel.repeat_interleave(hd, 1) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def token(x, u, t, top_k, top_p, min_p):
    """One row: the token by the definition, in plain Python floats (math.fsum for every sum)."""
    top_p, min_p, u = (off if math.isnan(v) else v for v, off in ((top_p, 1.0), (min_p, 0.0), (u, 0.0)))
    x = [float("-inf") if math.isnan(v) else float(v) for v in x]
    top = max(x)
    if top == float("-inf"):
        return 0
    if not t > 0:
        return x.index(top)
    w = [1.0 if v == top else (0.0 if math.isinf(v) or math.isinf(top) else math.exp((v - top) / max(t, 1e-30))) for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        want, n, run = max(top_p, 0.0) * math.fsum(w[i] for i in order), 0, 0.0
        while n < len(order) and (n == 0 or run < want):
            run += w[order[n]]
            n += 1
        order = order[:n]
    kept = sorted(i for i in order if w[i] >= min(min_p, 1.0))
    want, run = u * math.fsum(w[i] for i in kept), 0.0
    for i in kept:
        run += w[i]
        if run > want:
            return i
    return kept[-1]
