"""The 8-bit cache, forked prompts and draws with given numbers through the engine, as a server uses them together."""
import types

import pytest
import torch

from dlti_b200.models.config import PRESETS
from dlti_b200.models.llama import ResidentWeights
from dlti_b200.ops import kv8, rng
from dlti_b200.ops import serving as S
from dlti_b200.serve import model_runner
from dlti_b200.serve.engine import LLMEngine
from dlti_b200.serve.kv_cache import BlockManager, KVCache, KVCache8, KVSpec
from dlti_b200.serve.model_runner import TPContext, TPWeights
from dlti_b200.serve.params import Request, SamplingParams
from dlti_b200.serve.tokenizer import ByteTokenizer
from . import ref_cache8 as R

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def engine(dev="cpu", cfg="tiny-gqa", graphs=False, vocab=None, **kw):
    import copy
    cfg = copy.deepcopy(PRESETS[cfg])
    if vocab:
        cfg.vocab_size = vocab
    dt = torch.bfloat16 if dev == "cuda" else torch.float32
    full = ResidentWeights.random_init(cfg, dev, dt, seed=3)
    for t in full.all_matrices():
        t.mul_(4.0)
    w = TPWeights(cfg, 0, 1, dev, dt).load_from_full(full)
    kw = {"num_blocks": 64, "max_model_len": 256, "use_cuda_graphs": graphs} | kw
    return LLMEngine(cfg, w, TPContext(), ByteTokenizer(cfg.vocab_size), **kw)


def prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [[1] + torch.randint(3, 900, (n - 1,), generator=g).tolist() for n in lens]


def drain(eng):
    while eng.has_unfinished():
        eng.step()


# ---- 8-bit pages -----------------------------------------------------------------------------------------------------------------
def by_the_rules():
    """The ops of the 8-bit cache as tests/ref_cache8.py has them, on the host."""
    def rows(qkv, pos, cos, sin, slots, k8, v8, ks, vs, H, KV, hd):
        x = R.rotate(qkv.cpu().double(), pos.cpu().long(), cos.cpu().to(qkv.dtype).double(), sin.cpu().to(qkv.dtype).double(), H + KV, hd).to(qkv.dtype)
        for part, q, s in ((x[:, H * hd:(H + KV) * hd], k8, ks), (x[:, (H + KV) * hd:], v8, vs)):
            rq, rs = q.cpu().double(), s.cpu().double()
            R.write(part.double().view(-1, KV, hd), slots.cpu(), rq, rs)
            q.copy_(rq.float().to(torch.float8_e4m3fn))
            s.copy_(rs)
        return qkv.copy_(x)

    def acc(a, dtype, *args):
        out = rows(a.to(dtype), *args)
        a.zero_()
        return out

    def decode(q, k8, v8, ks, vs, tables, ctx, H, KV, hd, scale, out=None, max_ctx=None):
        o = R.attend(q.cpu(), k8.cpu(), v8.cpu(), ks.cpu(), vs.cpu(), tables.cpu(), ctx.cpu(), H, KV, hd, scale)[0].to(q.dtype).to(q.device)
        return o if out is None else out.copy_(o)

    return types.SimpleNamespace(rope_cache8_=rows, acc_rope_cache8=acc, paged_decode8=decode, gather_rows8_=kv8.gather_rows8_ref)


def logits_of(eng, seqs, chunk):
    """Logits of all tokens: each sequence enters `chunk` tokens at a time, then one by one; all in the same steps."""
    rs = [Request(f"r{i}", [], SamplingParams()) for i in range(len(seqs))]
    out, at = [], [0] * len(seqs)
    while any(a < len(s) for a, s in zip(at, seqs)):
        entries = []
        for i, (r, s) in enumerate(zip(rs, seqs)):
            n = min(chunk[i] if at[i] < len(s) - 6 else 1, len(s) - at[i])
            if n:
                entries.append((r, s[at[i]:at[i] + n], list(range(n))))
                at[i] += n
        out.append(eng.replay_step(entries))
    for r in rs:
        eng.replay_end(r)
    return torch.cat(out)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bs", [8, 16])
def test_engine_keeps_the_rules(dev, bs, monkeypatch):
    """Portions, single tokens and mixed steps over 8-bit pages: the logits are those of the same engine with the cache's rules in double precision.
    Two layers, whose outputs may round to the other neighbour in the compute type (2^-8 in bf16, 2^-24 sums in fp32 and, as a rounded key that falls
    on the other side of a border, 2^-4 of one number in some thousand): 2^-6 of the norm on the GPU, 2^-10 in fp32."""
    seqs = prompts([40, 9, 70, 23])
    got = logits_of(engine(dev, block_size=bs, kv_cache_dtype="fp8"), seqs, [16, 3, 70, 5])
    monkeypatch.setattr(model_runner, "K8", by_the_rules())
    eng = engine(dev, block_size=bs, kv_cache_dtype="fp8")
    want = logits_of(eng, seqs, [16, 3, 70, 5])
    assert eng.blocks.num_free == eng.blocks.num_blocks
    d = (got - want).norm(dim=1) / want.norm(dim=1)
    assert float(d.max()) < (2.0 ** -6 if dev == "cuda" else 2.0 ** -10)
    monkeypatch.undo()
    plain = logits_of(engine(dev, block_size=bs), seqs, [16, 3, 70, 5])
    assert float((got - plain).norm() / plain.norm()) > 2.0 ** -9            # it is not the 16-bit cache that ran


@pytest.mark.parametrize("kw", [dict(), dict(prefill_chunk=16, max_num_batched_tokens=40), dict(num_blocks=14), dict(mixed_batches=False),
                                dict(async_scheduling=False), dict(enable_prefix_caching=True)])
def test_generation_with_8_bits(kw):
    """Through the scheduler: chunked, preempted, prefix-cached; every page comes back."""
    eng = engine(kv_cache_dtype="fp8", **kw)
    ps = prompts([30, 61, 5, 47])
    out = eng.generate(ps, SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True))
    assert [len(o["token_ids"]) for o in out] == [12] * 4
    assert eng.blocks.num_free == eng.blocks.num_blocks and not any(eng.blocks.ref)
    assert isinstance(eng.kv, KVCache8) and KVCache8.bytes_per_block(2, 16, 2, 128) == 2 * 2 * 2 * (16 * 128 + 4)


def test_refusals():
    from dlti_b200.models.config import resolve_config
    from dlti_b200.models.registry import family_of
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        engine(kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="multiple of 8"):
        engine(kv_cache_dtype="fp8", block_size=4)
    cfg = resolve_config("sigosun-tiny")
    w = family_of(cfg).random_weights(cfg, "cpu", torch.float32, 0)
    for kw in (dict(kv_cache_dtype="fp8"), dict(fork_samples=True)):
        with pytest.raises(ValueError, match=cfg.name):
            LLMEngine(cfg, w, TPContext(), ByteTokenizer(cfg.vocab_size), num_blocks=16, max_num_seqs=2, max_model_len=64, **kw)
    for bad in (-0.1, 1.5):
        with pytest.raises(ValueError):
            SamplingParams(min_p=bad)


# ---- forks -----------------------------------------------------------------------------------------------------------------------
def test_block_manager_forks():
    bm = BlockManager(6, 4)
    a = []
    assert bm.ensure(a, 11)
    b, copies = bm.fork(a, 10)                               # two full blocks are shared, the third is copied
    assert b[:2] == a[:2] and copies == [(a[2], b[2])] and b[2] not in a and bm.num_free == 2
    c, copies = bm.fork(a, 8)
    assert c == a[:2] and copies == [] and [bm.ref[x] for x in a] == [3, 3, 1]
    d, _ = bm.fork(b, 9)
    assert bm.ensure(d, 12) and bm.num_free == 1 and bm.ensure(c, 12) and bm.num_free == 0
    assert bm.fork(a, 3) is None and bm.fork(a, 0) == ([], []) and [bm.ref[x] for x in a] == [4, 4, 1]
    for t in (a, c, b):
        bm.release(t)
    assert bm.num_free == 3 and bm.ref[d[0]] == 1            # the last one keeps what was shared
    bm.release(d)
    assert bm.num_free == 6 and not any(bm.ref)


def answers(eng, p, n, params=None, extra=()):
    """n answers to prompt p, asked for as the API does, beside other requests."""
    base = params or SamplingParams(max_tokens=10, temperature=0.0, ignore_eos=True)
    rids = []
    for i in range(n):
        sp = SamplingParams(**{**vars(base), "seed": 100 + i, "fork_of": "a-0" if i else None})
        rids.append(eng.add_request(list(p), sp, f"a-{i}"))
    for j, q in enumerate(extra):
        rids.append(eng.add_request(list(q), SamplingParams(**{**vars(base), "seed": 7 + j}), f"x-{j}"))
    drain(eng)
    return [list(eng.requests[r].output_ids) for r in rids]


@pytest.mark.parametrize("kw", [dict(), dict(prefill_chunk=16, max_num_batched_tokens=40), dict(mixed_batches=False), dict(async_scheduling=False),
                                dict(enable_prefix_caching=True), dict(num_blocks=13), dict(max_num_seqs=3)])
@pytest.mark.parametrize("length", [33, 32, 48, 2, 61])
def test_forked_answers_are_those_of_their_own_prompts(kw, length):
    """Greedy and drawn answers of forked requests are the ones that requests of their own give; the prompt runs once; every page comes back."""
    p, extra = prompts([length], length)[0], prompts([20, 7], 5)
    for base in (SamplingParams(max_tokens=10, temperature=0.0, ignore_eos=True), SamplingParams(max_tokens=10, temperature=0.9, top_p=0.9, ignore_eos=True)):
        one = engine(**kw)
        want = answers(one, p, 4, base, extra)
        eng = engine(fork_samples=True, **kw)
        got = answers(eng, p, 4, base, extra)
        assert got == want
        assert eng.blocks.num_free == eng.blocks.num_blocks and not any(eng.blocks.ref)
        if kw == {}:
            assert eng.sched.num_forks == 3 and eng.stats["prompt_tokens"] == length + 27 and one.sched.num_forks == 0


def test_forks_of_8_bit_pages_draw_with_given_numbers():
    """The three together: a prompt in 8-bit pages, answers that go on from copies of its last page, tokens drawn with min-p. Forks of the same
    seed agree whatever runs beside them."""
    p = prompts([45], 3)[0]
    base = SamplingParams(max_tokens=12, temperature=1.2, min_p=0.02, top_p=0.95, ignore_eos=True)
    eng = engine(fork_samples=True, kv_cache_dtype="fp8")
    first = answers(eng, p, 4, base)
    assert eng.sched.num_forks == 3 and eng.stats["prompt_tokens"] == 45 and len({tuple(a) for a in first}) == 4
    again = answers(engine(fork_samples=True, kv_cache_dtype="fp8"), p, 4, base, prompts([20, 7], 5))
    assert again[:4] == first


def test_fork_of_what_is_gone_or_differs():
    """An origin that ended, never was, or had another prompt: the request runs its own prompt."""
    p, q = prompts([20, 20], 1)
    eng = engine(fork_samples=True)
    sp = SamplingParams(max_tokens=4, temperature=0.0, ignore_eos=True)
    want = engine().generate([p, q], sp)
    eng.generate([p], sp)
    for prompt, origin, tokens in ((p, "nobody", want[0]), (q, "there", want[1]), (p, "self", want[0])):
        eng.add_request(list(p), SamplingParams(**vars(sp)), "there")
        rid = eng.add_request(list(prompt), SamplingParams(**{**vars(sp), "fork_of": origin}), "self")
        drain(eng)
        assert eng.requests[rid].output_ids == tokens["token_ids"]
    assert eng.sched.num_forks == 0 and eng.blocks.num_free == eng.blocks.num_blocks
    # an abort of the origin leaves its forks their pages
    eng.add_request(list(p), SamplingParams(max_tokens=30, temperature=0.0, ignore_eos=True), "o")
    rid = eng.add_request(list(p), SamplingParams(**{**vars(sp), "fork_of": "o"}), "f")
    for _ in range(3):
        eng.step()
    assert eng.sched.num_forks == 1
    eng.abort("o")
    drain(eng)
    assert eng.requests[rid].output_ids == want[0]["token_ids"] and eng.blocks.num_free == eng.blocks.num_blocks


def test_copies_reach_every_layer_once():
    """Layers of different shapes, layers that share another's pages, layers without any."""
    kv = KVCache.from_specs([KVSpec(2, 8, 4), None, KVSpec(1, 16, 0), KVSpec(2, 8, 4, source=0)], 5, 4, torch.float32, "cpu")
    for i, t in enumerate(t for t in (*kv.k, *kv.v) if t is not None):
        t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(i)))
    k0, k2 = kv.k[0].clone(), kv.k[2].clone()
    kv.copy_pages([1, 3], [4, 0])
    assert torch.equal(kv.k[0][4], k0[1]) and torch.equal(kv.k[2][0], k2[3]) and torch.equal(kv.k[0][1:4], k0[1:4]) and kv.k[3] is kv.k[0]


def test_answers_of_the_api():
    pytest.importorskip("fastapi")
    from fastapi.testclient import TestClient

    from dlti_b200.serve.api_server import AsyncEngine, _answer, _params_from_body, build_app
    sp = SamplingParams(n=3)
    assert [_answer(sp, "c", i).fork_of for i in range(6)] == [None, "c-0", "c-0", None, "c-3", "c-3"] and sp.fork_of is None
    assert _params_from_body({"min_p": 0.1}).min_p == 0.1
    eng = engine(fork_samples=True, kv_cache_dtype="fp8")
    aeng = AsyncEngine(eng)
    aeng.start()
    try:
        with TestClient(build_app(aeng, "tiny")) as c:
            ask = {"prompt": [prompts([40], 1)[0], prompts([25], 2)[0]], "max_tokens": 8, "n": 3, "temperature": 0.8, "min_p": 0.05, "ignore_eos": True, "seed": 4}
            j = c.post("/v1/completions", json=ask).json()
            assert len(j["choices"]) == 6 and j["usage"]["completion_tokens"] == 48
            assert c.post("/v1/completions", json={**ask, "min_p": 2}).status_code == 400
            j = c.post("/v1/chat/completions", json={"messages": [{"role": "user", "content": "hello there, machine"}], "n": 2, "max_tokens": 8, "temperature": 0, "ignore_eos": True}).json()
            assert len(j["choices"]) == 2
    finally:
        aeng.stop = True
        aeng.thread.join(timeout=10)
    assert eng.sched.num_forks == 5 and eng.blocks.num_free == eng.blocks.num_blocks


# ---- draws -----------------------------------------------------------------------------------------------------------------------
def test_uniforms():
    """53 bits, a function of the seed alone, evenly spread."""
    a = rng.uniforms(list(range(4000)) + [2 ** 63 - 1])
    assert a.min() >= 0 and a.max() < 1 and len(set(a.tolist())) == 4001 and abs(a.mean() - 0.5) < 0.02 and (a * 2.0 ** 53 == (a * 2.0 ** 53).round()).all()
    assert rng.uniforms([17]).tolist() == [a[17]]


@pytest.mark.parametrize("dev", DEVICES)
def test_min_p_draws(dev):
    """A min-p of 1 leaves the likeliest token; steps in which nobody asks for it draw as before; others draw with the numbers of their seeds."""
    ps = prompts([12, 30], 2)
    sp = dict(max_tokens=8, ignore_eos=True, seed=5)
    eng = engine(dev)
    seen = []
    def spy(logits, u, *a, **kw):
        tok, lp = S.sample_given(logits, u, *a, **kw)
        seen.append((logits.float().cpu(), u.cpu().clone(), [x.cpu().clone() for x in a], tok.cpu().clone()))
        return tok, lp
    import dlti_b200.serve.engine as E
    real = E.S
    E.S = types.SimpleNamespace(**{**vars(S), "sample_given": spy})
    try:
        eng.generate(ps, SamplingParams(temperature=2.0, **sp))
        assert not seen
        eng.generate(ps, [SamplingParams(temperature=2.0, min_p=1.0, **sp), SamplingParams(temperature=1.5, min_p=0.05, top_k=30, **sp)])
    finally:
        E.S = real
    assert len(seen) >= 8
    for lg, u, (t, k, p, m), tok in seen:
        for b in range(len(tok)):
            assert int(tok[b]) == R.token(lg[b].double().tolist(), float(u[b]), float(t[b]), int(k[b]), float(p[b]), float(m[b]))
    assert all(int(tok[0]) == int(lg[0].argmax()) for lg, _, (t, k, p, m), tok in seen if float(m[0]) == 1.0)


@pytest.mark.gpu
def test_large_vocabulary():
    """More logits than `sample` holds on a GPU (it refuses them): the engine draws with given numbers, greedy and not, replayed graphs included."""
    eng = engine("cuda", vocab=60032, graphs=True)
    ps = prompts([12, 30, 5], 2)
    out = eng.generate(ps, SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True))
    again = engine("cuda", vocab=60032).generate(ps, SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True))
    assert [o["token_ids"][0] for o in out] == [o["token_ids"][0] for o in again]
    drawn = eng.generate(ps, SamplingParams(max_tokens=6, temperature=1.0, top_p=0.9, ignore_eos=True, seed=3))
    assert all(0 <= t < 60032 for o in drawn for t in o["token_ids"]) and eng.graphs


@pytest.mark.gpu
def test_replayed_and_eager_steps_agree(monkeypatch):
    """8-bit pages, forks and min-p in captured decode steps: the tokens of eager ones."""
    import dlti_b200.ops.gemm as G
    monkeypatch.setattr(G, "_SKINNY_SPLIT", 1)               # a summation order that does not change from run to run
    p = prompts([45], 3)[0]
    base = SamplingParams(max_tokens=16, temperature=1.2, min_p=0.02, ignore_eos=True)
    kw = dict(fork_samples=True, kv_cache_dtype="fp8")
    got = [answers(engine("cuda", graphs=g, **kw), p, 4, base, prompts([20, 7], 5)) for g in (True, False)]
    assert got[0] == got[1]
