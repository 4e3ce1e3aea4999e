"""The order in which forks and other requests get pages."""
import pytest

from dlti_b200.serve.kv_cache import BlockManager
from dlti_b200.serve.params import Request, SamplingParams
from dlti_b200.serve.scheduler import Scheduler


def req(rid, n, tokens, fork_of=None):
    return Request(rid, list(range(n)), SamplingParams(max_tokens=tokens, fork_of=fork_of))


def step(s):
    """One step, whose tokens are read at once. The ids of what ran in it."""
    b = s.schedule()
    if b is None:
        return []
    for r in b.requests[b.num_decode:]:
        r.num_computed += r.chunk
    for r in b.requests[:b.num_sampled]:
        r.prefill_done = True
        r.output_ids.append(1)
        if len(r.output_ids) >= r.params.max_tokens:
            s.finish(r, "length")
    return [r.request_id for r in b.requests]


@pytest.mark.parametrize("chunk", [0, 8])
def test_a_fork_is_not_kept_from_its_pages(chunk):
    """Pages come free one at a time while short requests keep arriving, and a fork needs two: those that came after it wait until it has them."""
    s = Scheduler(BlockManager(5, 16), max_num_seqs=8, max_num_batched_tokens=64, max_model_len=48, prefill_chunk=chunk, fork_samples=True)
    s.add(req("o", 16, 14))
    for i in range(3):
        s.add(req(f"x{i}", 2, i + 3))
    while not any(r.request_id == "o" and r.output_ids for r in s.running):
        step(s)
    s.add(req("f", 16, 2, fork_of="o"))
    ran = []
    for i in range(8):
        s.add(req(f"y{i}", 2, 3))
        ran.append(step(s))
    first = next((i for i, r in enumerate(ran) if "f" in r), None)
    assert first is not None and not any(x.startswith("y") for r in ran[:first] for x in r)
    assert s.num_forks == 1 and s.num_preemptions == 0
    for _ in range(60):
        step(s)
    assert not s.has_work() and s.blocks.num_free == 5 and not any(s.blocks.ref)


def test_forks_pass_prompts_that_wait_for_pages():
    """A prompt that needs more pages than are free does not keep back the answers of a request that runs: their pages are there only as long as it
    does. It is next when it ends, before any later prompt."""
    s = Scheduler(BlockManager(8, 4), max_num_seqs=8, max_num_batched_tokens=64, max_model_len=32, fork_samples=True)
    s.add(req("o", 8, 6))
    step(s)
    for r in (req("big", 23, 2), req("f", 8, 3, fork_of="o"), req("late", 2, 2)):
        s.add(r)
    seen = [step(s) for _ in range(20)]
    when = {n: next(i for i, r in enumerate(seen) if n in r) for n in ("big", "f", "late")}
    assert when["f"] == 0 and when["f"] < when["big"] <= when["late"] and not s.has_work() and s.blocks.num_free == 8
