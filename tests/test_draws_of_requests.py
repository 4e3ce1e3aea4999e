"""What a request draws is its own matter: its seed, its settings and its place among the answers to a prompt, not what runs beside it."""
import json
import os
import socket
import subprocess
import sys

import pytest

from dlti_b200.serve.params import SamplingParams
from .test_cache8_serving import DEVICES, engine, prompts


def run(eng, requests, late=4):
    """requests: (id, prompt, params, whether it joins after `late` steps). The tokens and log-probabilities of each."""
    for rid, p, sp, _ in (r for r in requests if not r[3]):
        eng.add_request(list(p), sp, rid)
    for _ in range(late):
        eng.step()
    for rid, p, sp, _ in (r for r in requests if r[3]):
        eng.add_request(list(p), sp, rid)
    while eng.has_unfinished():
        eng.step()
    return {r[0]: (list(eng.requests[r[0]].output_ids), list(eng.requests[r[0]].logprobs)) for r in requests}


@pytest.mark.parametrize("graphs", [False, pytest.param(True, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("mine", [0.0, 0.03])
def test_a_seeded_request_beside_neighbours(dev, graphs, mine, monkeypatch):
    """A request with or without min-p, beside a neighbour that joins late, ends early, and has min-p or not: the same tokens and log-probabilities."""
    import dlti_b200.ops.gemm as G
    monkeypatch.setattr(G, "_SKINNY_SPLIT", 1)               # a summation order that does not change from run to run
    if graphs and dev == "cpu":
        pytest.skip("graphs are captured on a GPU")
    p, q = prompts([12, 30], 2)
    got = []
    for theirs in (0.0, 1e-50, 0.05, 1.0):                   # (1e-50 is none in the 32 bits that a row has for it)
        a = SamplingParams(max_tokens=20, temperature=1.5, top_p=0.95, min_p=mine, seed=5, ignore_eos=True, logprobs=1)
        b = SamplingParams(max_tokens=7, temperature=0.0, min_p=theirs, ignore_eos=True)
        got.append(run(engine(dev, graphs=graphs), [("a", p, a, False), ("b", q, b, True)]))
    assert len(got[0]["a"][0]) == 20 and len(set(got[0]["a"][0])) > 3
    for g in got[1:]:
        assert g["a"] == got[0]["a"] and g["b"][0] == got[0]["b"][0]


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_of_both_kinds_in_one_step(dev, monkeypatch):
    """Requests with min-p between others without, drawn and greedy: each has the tokens that it has where all are of one kind in its step."""
    import dlti_b200.ops.gemm as G
    monkeypatch.setattr(G, "_SKINNY_SPLIT", 1)
    ps = prompts([12, 30, 5, 21], 3)
    sps = [SamplingParams(max_tokens=8, temperature=t, min_p=m, top_k=40, seed=9 + i, ignore_eos=True)
           for i, (t, m) in enumerate(((1.2, 0.0), (1.4, 0.02), (0.0, 0.0), (0.0, 0.3)))]

    def take(change):
        out = engine(dev, async_scheduling=False).generate(ps, [SamplingParams(**{**vars(s), **change(s)}) for s in sps])
        return [o["token_ids"] for o in out]

    mixed = take(lambda s: {})
    off = take(lambda s: {"min_p": 0.0})                     # as many rows of the same prompts, all by `sample`
    on = take(lambda s: {"min_p": s.min_p or 0.02})          # and all by `sample_given`
    assert [mixed[0], mixed[1], mixed[2], mixed[3]] == [off[0], on[1], off[2], on[3]] and mixed[0] != on[0] and mixed[1] != off[1]


TWO = r"""
import json, sys, torch
sys.path.insert(0, {root!r})
from dlti_b200.models.config import PRESETS
from dlti_b200.parallel import comm
from dlti_b200.serve.engine import LLMEngine
from dlti_b200.serve.model_runner import TPContext, TPWeights
from dlti_b200.serve.params import SamplingParams
from dlti_b200.serve.tokenizer import ByteTokenizer
info = comm.init_distributed("cpu")
cfg = PRESETS["tiny"]
w = TPWeights(cfg, info.rank, info.world_size, "cpu", torch.float32).init_random(5)
for l in w.layers:
    for k in ("w_qkv", "w_o", "w_gu", "w_down"):
        l[k].mul_(4.0)
w.embed.mul_(4.0); w.lm_head.mul_(4.0)
eng = LLMEngine(cfg, w, TPContext(info, "nccl", None, cfg), ByteTokenizer(cfg.vocab_size), info=info, num_blocks=20, max_model_len=256, use_cuda_graphs=False)
if info.rank != 0:
    eng.worker_loop()
else:
    sps = [SamplingParams(max_tokens=n, temperature=1.3, min_p=m, seed=3, ignore_eos=True, logprobs=1) for n, m in ((12, 0.0), (6, 0.04), (9, 0.0))]
    out = eng.generate([[1] + list(range(40, 40 + n)) for n in (5, 33, 20)], sps)
    eng.shutdown_workers()
    json.dump([o["token_ids"] for o in out], open(sys.argv[1], "w"))
comm.shutdown()
"""


@pytest.mark.parametrize("control", ["shm", "gloo"])
def test_steps_of_both_kinds_on_two_ranks(tmp_path, control):
    """Every rank draws a step's rows the same way (gloo, two processes): the tokens of one process."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = tmp_path / "two.py"
    script.write_text(TWO.format(root=root))
    env = dict(os.environ, PYTHONPATH=root, OMP_NUM_THREADS="2", DLTI_TP_CONTROL=control)
    out = []
    for world in (1, 2):
        to = tmp_path / f"{world}.json"
        cmd, e = [sys.executable, str(script), str(to)], dict(env, WORLD_SIZE="1", RANK="0", LOCAL_RANK="0")
        if world == 2:
            with socket.socket() as so:
                so.bind(("127.0.0.1", 0))
                port = so.getsockname()[1]
            cmd, e = [sys.executable, "-m", "dlti_b200.launch", "--num_gpus=2", f"--master_port={port}", "--no_local_rank", str(script), str(to)], env
        r = subprocess.run(cmd, env=e, capture_output=True, text=True, timeout=300, cwd=root)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
        out.append(json.load(open(to)))
    assert out[0] == out[1] and [len(t) for t in out[0]] == [12, 6, 9]


def test_answers_to_one_seeded_prompt():
    """Through the API: with a seed, the n answers of a request with min-p differ from one another, repeat from call to call, and the first one is
    the answer to n = 1. Streams and chats, too."""
    pytest.importorskip("fastapi")
    from fastapi.testclient import TestClient

    from dlti_b200.serve.api_server import AsyncEngine, build_app
    eng = engine(fork_samples=True)
    aeng = AsyncEngine(eng)
    aeng.start()
    try:
        with TestClient(build_app(aeng, "tiny")) as c:
            def texts(**more):
                ask = {"prompt": prompts([20, 9], 1), "max_tokens": 8, "n": 3, "temperature": 1.5, "min_p": 0.02, "ignore_eos": True, "seed": 4, **more}
                chat = more.pop("chat", None)
                if chat:
                    ask = {"messages": [{"role": "user", "content": "hello"}], **{k: v for k, v in ask.items() if k not in ("prompt", "chat")}}
                r = c.post("/v1/chat/completions" if chat else "/v1/completions", json=ask)
                out = {}
                if more.get("stream"):
                    parts = [json.loads(x[6:]) for x in r.text.split("\n\n") if x.startswith("data: {")]
                else:
                    parts = [r.json()]
                for ch in (ch for part in parts for ch in part["choices"]):
                    out[ch["index"]] = out.get(ch["index"], "") + (ch.get("text") or (ch.get("message") or ch.get("delta") or {}).get("content") or "")
                return [out[i] for i in sorted(out)]

            first = texts()
            assert len(set(first)) == 6 and texts() == first and texts(stream=True) == first
            assert texts(n=1) == first[::3] and texts(seed=5) != first
            talk = texts(chat=True)
            assert len(set(talk)) == 3 and texts(chat=True, stream=True) == talk and texts(chat=True, n=1) == talk[:1]
    finally:
        aeng.stop = True
        aeng.thread.join(timeout=10)
    assert eng.sched.num_forks > 0


@pytest.mark.parametrize("dev,vocab,min_p", [("cpu", None, 0.02), pytest.param("cuda", None, 0.02, marks=pytest.mark.gpu),
                                             pytest.param("cuda", 60032, 0.0, marks=pytest.mark.gpu)])
def test_places_among_the_answers(dev, vocab, min_p):
    """One seed, four places: four texts, also where a long vocabulary is what brings the numbers; a place is none of its row's."""
    p = prompts([14], 4)[0]
    sp = [SamplingParams(max_tokens=10, temperature=1.5, min_p=min_p, seed=2 ** 62 + 7, answer=i, ignore_eos=True) for i in range(4)]
    got = engine(dev, vocab=vocab, max_num_seqs=8).generate([p] * 4, sp)
    assert len({tuple(o["token_ids"]) for o in got}) == 4
    with pytest.raises(ValueError):
        SamplingParams(answer=-1)
    if dev == "cpu":
        back = engine(dev).generate([p] * 4, sp[::-1])
        assert [o["token_ids"] for o in back[::-1]] == [o["token_ids"] for o in got]


def test_numbers_of_a_seed():
    from dlti_b200.ops.rng import uniforms
    s = list(range(500)) + [2 ** 63 - 1]
    a = [uniforms(s, i).tolist() for i in range(5)]
    assert a[0] == uniforms(s).tolist() and len({x for r in a for x in r}) == 5 * 501
    assert uniforms([3, 3, 9], [0, 4, 1]).tolist() == [a[0][3], a[4][3], a[1][9]]


@pytest.mark.parametrize("dev", DEVICES)
def test_vocabularies_that_no_sampler_holds(dev):
    """More logits than a row can be drawn from: a request is refused when it comes, not in the engine's next step, and nothing of it stays. On the
    host that is so for requests with min-p. Replays, which draw nothing, go on."""
    from dlti_b200.serve.params import Request
    eng = engine(dev, vocab=262144 + 64)
    p = prompts([5], 1)[0]
    for m in (0.1, 0.0) if dev == "cuda" else (0.1,):
        with pytest.raises(ValueError, match="262144"):
            eng.add_request(p, SamplingParams(min_p=m), "r")
    assert not eng.has_unfinished() and not eng.requests
    if dev == "cpu":
        assert len(eng.generate([p], SamplingParams(max_tokens=2, temperature=1.0, seed=1, ignore_eos=True))[0]["token_ids"]) == 2
    assert eng.replay_step([(Request("s", [], SamplingParams()), p, [4])]).shape == (1, 262144 + 64)


@pytest.mark.gpu
def test_the_longest_vocabulary():
    eng = engine("cuda", vocab=262144, graphs=True)
    out = eng.generate(prompts([5, 9], 1), [SamplingParams(max_tokens=4, temperature=t, min_p=0.001, seed=1, ignore_eos=True) for t in (0.0, 1.0)])
    assert all(len(o["token_ids"]) == 4 and max(o["token_ids"]) < 262144 for o in out)


def test_sampling_parameters_by_place():
    """Their order, for calls that give them by place: what came later comes last."""
    import dataclasses
    names = [f.name for f in dataclasses.fields(SamplingParams)]
    assert names[:14] == ["max_tokens", "temperature", "top_p", "top_k", "n", "seed", "stop", "stop_token_ids", "ignore_eos", "min_tokens", "logprobs", "echo",
                          "skip_special_tokens", "detokenize"]
    sp = SamplingParams(8, 0.7, 0.9, 40, 1, 42, ["x"])
    assert (sp.n, sp.seed, sp.stop, sp.min_p) == (1, 42, ["x"], 0.0)


def test_settings_of_a_packed_step():
    """With and without min-p and places, as pack_step takes them."""
    from dlti_b200.ops.rng import uniforms
    eng = engine()
    row = ([0.7, 0.0], [0, 3], [1.0, 0.5], [11, 12])
    pack = lambda *more: eng.pack_step(2, [4, 5], [0, 0], [0, 16], [1, 1], [[0], [1]], [], 0, (*row, *more))
    assert [pack(*m).layout.given for m in ((), ([0.0, 0.0],), ([0.1, 0.0],), ([0.1, 0.2],), ([0.1, 1e-50], [0, 2]))] == [0, 0, 2, 1, 2]
    import numpy as np
    for more, want in ((([0.1, 0.0],), uniforms([11, 12])), (([0.1, 0.0], [3, 1]), uniforms([11, 12], [3, 1]))):
        step = pack(*more)
        v = step.layout.views(step.slot[0].numpy(), np)
        assert v["unif"].tolist() == want.tolist() and v["minp"].tolist() == [np.float32(0.1), 0.0] and v["seeds"].tolist() == row[3]
