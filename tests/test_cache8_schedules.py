"""What 8-bit pages hold while the scheduler moves requests about: chunked, preempted, prefix-cached, forked.

Keys and values of the first layer follow from a token and its position alone, so every cached row can be compared with them, in double precision."""
import copy

import pytest
import torch

from dlti_b200.ops.elementwise import rope_tables
from dlti_b200.serve import model_runner
from dlti_b200.serve.params import SamplingParams
from . import ref_cache8 as R
from .test_cache8_serving import DEVICES, by_the_rules, engine, prompts


def first_layer(eng, tokens):
    """(keys and values [2, n, KV, hd] of the tokens at positions 0 .., how far off the engine's may be) in float64."""
    cfg, w = eng.cfg, eng.w
    hd, H, KV, n, dt = cfg.head_dim, w.H, w.KV, len(tokens), w.embed.dtype
    x = w.embed.cpu().double()[tokens]
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + cfg.rms_norm_eps) * w.layers[0]["ln1"].cpu().double()
    m = w.layers[0]["w_qkv"].cpu().double()[H * hd:]
    y, size = x @ m.T, x.abs() @ m.abs().T
    cos, sin = (t[:n].to(dt).double() for t in rope_tables(cfg.max_position_embeddings, hd, cfg.rope_theta, "cpu"))
    k = R.rotate(y[:, :KV * hd], torch.arange(n), cos, sin, KV, hd)
    a = size[:, :KV * hd].view(n, KV, 2, hd // 2)
    size = torch.cat([(a.sum(2, keepdim=True).expand_as(a)).reshape(n, -1), size[:, KV * hd:]], 1)
    # roundings of the normalised row, of the product and of the rotation, of half a step each (eps / 2); in fp32 sums of 256 products besides
    off = 4 * torch.finfo(dt).eps * size + 256 * 2.0 ** -24 * size
    return torch.cat([k, y[:, KV * hd:]], 1).view(n, 2, KV, hd).transpose(0, 1), off.view(n, 2, KV, hd).transpose(0, 1)


def cached(eng, r):
    """Rows of r that are in the cache and whose tokens the host knows."""
    n = r.sched_tokens - 1 if r.prefill_done else r.num_computed
    return (r.prompt_ids + r.output_ids)[:n]


def check(eng, own=True):
    """Every cached row of every running request. own: nobody else ever wrote into its pages, so that their scales are the smallest that fit."""
    bs, seen = eng.blocks.block_size, 0
    pages = [(q[0].cpu().double(), s[0].cpu().double()) for q, s in ((eng.kv.k, eng.kv.k_scale), (eng.kv.v, eng.kv.v_scale))]
    for r in eng.sched.running:
        tokens = cached(eng, r)
        if not tokens:
            continue
        want, off = first_layer(eng, tokens)
        at = torch.arange(len(tokens))
        page, place = torch.tensor(r.blocks)[at // bs], at % bs
        for (q, s), x, tol in zip(pages, want, off):
            held, scale = q[page, :, place] * s[page][..., None], s[page][..., None]
            # a row was rounded when it came (half of 2^-3 of it, or of the smallest step, 2^-9 scales) and, of the small numbers, when the scale
            # rose: to steps of which each is at least twice the last, so that all of them together are less than one of 2^-9 scales now
            assert bool(((held - x).abs() <= 2.0 ** -4 * (x.abs() + tol) + 2.0 ** -9 * scale + tol).all()), (r.request_id, len(tokens))
            for p in range(-(-len(tokens) // bs)):
                top, slack = x[p * bs:(p + 1) * bs].abs().amax((0, 2)), tol[p * bs:(p + 1) * bs].amax((0, 2))
                now = s[r.blocks[p]]
                assert bool((448 * now >= top - slack).all())
                # tokens in flight, which the host does not know, may have raised the last page
                if own and (p + 1) * bs <= len(tokens):
                    assert bool((now <= torch.tensor([R.scale_of(float(t)) for t in top + slack])).all())
        seen += len(tokens)
    return seen


KINDS = [dict(), dict(prefill_chunk=16, max_num_batched_tokens=40), dict(num_blocks=14), dict(num_blocks=14, prefill_chunk=16, max_num_batched_tokens=40),
         dict(mixed_batches=False), dict(async_scheduling=False), dict(enable_prefix_caching=True), dict(enable_prefix_caching=True, num_blocks=14), dict(enable_prefix_caching=True, num_blocks=10)]


def schedule(kw, ps, more, dev="cpu", watch=None, **other):
    """Four requests, and four more once the first of them have ended."""
    eng = engine(dev, kv_cache_dtype="fp8", **kw, **other)
    sp = SamplingParams(max_tokens=14, temperature=0.0, ignore_eos=True)
    ids = [eng.add_request(list(p), copy.copy(sp), f"r{i}") for i, p in enumerate(ps)]
    rows = 0
    while eng.has_unfinished():
        eng.step()
        rows += watch(eng) if watch else 0
        if more and any(eng.requests[i].status == "finished" for i in ids):
            ids += [eng.add_request(list(p), copy.copy(sp), f"s{i}") for i, p in enumerate(more)]
            more = ()
    return eng, rows, [eng.requests[i].output_ids for i in ids]


@pytest.mark.parametrize("graphs", [False, pytest.param(True, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kw", KINDS)
def test_rows_of_every_schedule(dev, graphs, kw):
    """All rows are where the block tables say, with scales that fit them: pages that are handed out again, that are shared, that are written in
    portions."""
    if graphs and dev == "cpu":
        pytest.skip("graphs are captured on a GPU")
    ps = prompts([30, 61, 5, 47])
    shared = [ps[1][:40] + t for t in prompts([9, 21], 8)] + prompts([52, 16], 9)
    eng, rows, out = schedule(kw, ps, shared, dev, check, graphs=graphs)
    assert rows > 2000 and all(len(t) == 14 for t in out)
    if "num_blocks" in kw and kw != dict(enable_prefix_caching=True, num_blocks=14):       # (there what is shared leaves room for all)
        assert eng.sched.num_preemptions > 0
    if kw.get("enable_prefix_caching"):
        assert eng.blocks.hits >= 32
    assert eng.blocks.num_free == eng.blocks.num_blocks and not any(eng.blocks.ref)


@pytest.mark.parametrize("kw", KINDS)
def test_logits_of_every_schedule(kw, monkeypatch):
    """The logits that tokens are taken from are those of the same schedule with the cache's rules in double precision: 2^-10 of their norm, as in
    test_cache8_serving.py, and the same tokens."""
    import dlti_b200.serve.engine as E
    ps = prompts([30, 61, 5, 47])
    shared = [ps[1][:40] + t for t in prompts([9], 8)]
    real, runs = E.S.sample, []

    def spy(logits, *a, **k):
        runs[-1].append(logits.clone())
        return real(logits, *a, **k)

    monkeypatch.setattr(E.S, "sample", spy)
    out = []
    for rules in (False, True):
        if rules:
            monkeypatch.setattr(model_runner, "K8", by_the_rules())
        runs.append([])
        out.append(schedule(kw, ps, shared)[2])
    assert out[0] == out[1] and len(runs[0]) == len(runs[1]) > 15
    for a, b in zip(*runs):
        assert float(((a - b).norm(dim=1) / b.norm(dim=1)).max()) < 2.0 ** -10


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("length", [45, 33, 32, 2])
@pytest.mark.parametrize("wait", [0, 9])
def test_rows_of_forks(dev, length, wait):
    """Forks at once, and forks of an origin that has gone on for some tokens: the copied page may have the scale that these gave it, no less than its
    rows need and no more than the origin's page, and its rows are what they were but for the smallest step of that scale."""
    p = prompts([length], 3)[0]
    eng = engine(dev, kv_cache_dtype="fp8", fork_samples=True)
    sp = dict(temperature=1.5, min_p=0.01, ignore_eos=True)
    eng.add_request(list(p), SamplingParams(max_tokens=wait + 18, seed=1, **sp), "o")
    for _ in range(wait):
        eng.step()
        check(eng)
    for i in range(3):
        eng.add_request(list(p), SamplingParams(max_tokens=6, seed=2 + i, fork_of="o", **sp), f"f{i}")
    bs, copied = eng.blocks.block_size, 0
    real = eng.kv.copy_pages

    def spy(src, dst):
        nonlocal copied
        real(src, dst)
        copied += len(dst)
        for s in (*eng.kv.k_scale, *eng.kv.v_scale):
            assert torch.equal(s[dst], s[src])

    eng.kv.copy_pages = spy
    rows = 0
    while eng.has_unfinished():
        eng.step()
        rows += check(eng, own=False)
    assert rows > 100 and eng.sched.num_forks == 3 and copied == (3 if (length - 1) % bs else 0)
    assert eng.blocks.num_free == eng.blocks.num_blocks and not any(eng.blocks.ref)
