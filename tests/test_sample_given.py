"""Tokens from given random numbers against the definition in plain Python sums (tests/ref_cache8.py token)."""
import math

import pytest
import torch

from dlti_b200.ops import serving as S
from . import ref_cache8 as R

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def run(x, u, t, k, p, m, dev, check_lp=True):
    """x [B, V]; settings: a number for all rows or one for each (None: not given)."""
    B = x.shape[0]
    full = lambda v, dt: None if v is None else torch.tensor([v] * B if not isinstance(v, list) else v, dtype=dt)
    T, K, P, M = full(t, torch.float32), full(k, torch.int32), full(p, torch.float32), full(m, torch.float32)
    to = lambda a: None if a is None else a.to(dev)
    tok, lp = S.sample_given(x.to(dev), to(u), to(T), to(K), to(P), to(M), want_logprob=True)
    tok, lp = tok.cpu(), lp.cpu()
    at = lambda a, b, off: off if a is None else float(a[b])
    want = [R.token(x[b].double().tolist(), float(u[b]), at(T, b, 0.0), int(at(K, b, 0)), at(P, b, 1.0), at(M, b, 0.0)) for b in range(B)]
    assert tok.tolist() == want
    if check_lp:
        ref = torch.log_softmax(x.double(), -1)[torch.arange(B), tok]
        # a difference of logits and a logarithm in fp32 (2^-23 of each), the sum of exponentials of 2 ulp each in fp32 sums of up to V / 1024 terms
        tol = 2.0 ** -22 * (1 + ref.abs()) + (x.shape[1] / 1024 + 8) * 2.0 ** -23
        assert bool(((lp.double() - ref).abs() <= tol).all())
    only, none = S.sample_given(x.to(dev), to(u), to(T), to(K), to(P), to(M))
    assert none is None and torch.equal(only.cpu(), tok)
    return tok


def uniform(B, seed):
    return torch.rand(B, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def logits(B, V, seed, sharp=2.5, dtype=torch.bfloat16):
    return (torch.randn((B, V), generator=torch.Generator().manual_seed(seed)) * sharp).to(dtype)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 300, 1024, 8192, 8193, 20001])
def test_settings(dev, dtype, V):
    B = 12
    x = logits(B, V, V, dtype=dtype)
    u = uniform(B, V + 1)
    t = [0.0, 1.0, 0.5, 1.5, 0.1, 5.0, 1.0, 1.0, 1.0, 0.7, 1.0, -1.0]
    k = [0, 0, 50, 1, 0, 1000, 5, 0, 3, 20, 100000, 4]
    p = [1.0, 1.0, 1.0, 1.0, 0.9, 0.95, 0.5, 0.0, 0.99, 0.3, 1.0, 0.5]
    m = [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.02, 0.0, 0.0, 0.2, 1.0, 0.5]
    run(x, u, t, k, p, m, dev)
    run(x, u, t, None, None, None, dev)
    run(x, u, None, k, p, m, dev)
    run(x, u, t, None, p, None, dev)
    run(x, u, t, k, None, None, dev)
    run(x, u, t, None, None, m, dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("seed", range(4))
def test_many_draws(dev, seed):
    """Different settings over many rows, flat and sharp."""
    B, V, g = 96, 3001, torch.Generator().manual_seed(seed)
    x = logits(B, V, seed + 10, 1.0) * torch.rand((B, 1), generator=g).mul(6).to(torch.bfloat16)
    pick = lambda xs: [xs[i] for i in torch.randint(0, len(xs), (B,), generator=g).tolist()]
    run(x, uniform(B, seed), pick([0.3, 0.7, 1.0, 1.3, 3.0]), pick([0, 0, 1, 2, 40, 500, 2999, 3001]), pick([1.0, 0.999, 0.95, 0.9, 0.5, 0.01]),
        pick([0.0, 0.0, 0.01, 0.1, 0.9]), dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [33, 1500, 9000, 20000])
def test_equal_logits(dev, V):
    """Ties go to the lowest index: all equal, two levels, zeros of both signs, more equal ones than a bin's list holds."""
    B = 8
    u = uniform(B, V)
    u[0], u[1] = 0.0, 1 - 2.0 ** -53
    k, p, m = [0, 5, 0, V // 2, 1, 0, 1300, 7], [1.0, 1.0, 0.5, 1.0, 1.0, 0.25, 0.5, 0.75], 0.0
    run(torch.full((B, V), 1.5, dtype=torch.bfloat16), u, 1.0, k, p, m, dev)
    two = torch.full((B, V), -1.0)
    two[:, ::3] = 2.0
    run(two.to(torch.float16), u, 0.8, k, p, m, dev)
    zero = torch.zeros((B, V))
    zero[:, 1::2] = -0.0
    run(zero, u, 1.0, k, p, m, dev)
    run(torch.full((B, V), 1.5, dtype=torch.bfloat16), u, 0.0, k, p, m, dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_narrow_and_wide_rows(dev):
    """Logits within 2^-20 of one another (one bin holds them all), and thousands apart (most weigh nothing)."""
    B, V = 8, 5000
    u, g = uniform(B, 1), torch.Generator().manual_seed(2)
    k, p, m = [0, 2000, 0, 1, 0, 2500, 50, 0], [1.0, 1.0, 0.5, 0.5, 0.001, 0.7, 0.9, 0.999], [0, 0, 0, 0, 0.5, 0, 0, 1.0]
    run(3 + torch.rand((B, V), generator=g) * 2.0 ** -20, u, 1.0, k, p, m, dev)
    run(torch.randn((B, V), generator=g) * 3000, u, 1.0, k, p, m, dev)
    run(torch.randn((B, V), generator=g), u, [1e-30, 1e-4, 1e30, 1e4, 1e-2, 100.0, 3e38, 1e-38], k, p, m, dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_masked_rows(dev):
    """-inf is never drawn while anything else is there, nor is NaN; +inf always is; the lowest number of the type is a number; a row with nothing
    left gives token 0."""
    B, V = 9, 2000
    x = logits(B, V, 3, dtype=torch.float32)
    x[0, :] = -math.inf
    x[1, :] = math.nan
    x[2, :1999] = -math.inf
    x[3, ::2] = math.nan
    x[4, 5] = x[4, 1000] = math.inf
    x[5, 10:] = torch.finfo(torch.float32).min
    x[6, :] = torch.finfo(torch.float32).min
    x[7, 3:] = -math.inf
    u = uniform(B, 4)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (1.0, 100, 0.9, 0.01), (0.0, 0, 1.0, 0.0), (2.0, 0, 0.5, 0.0), (math.inf, 0, 1.0, 0.0)):
        tok = run(x, u, t, k, p, m, dev, check_lp=False)
        assert tok[:3].tolist() == [0, 0, 1999] and tok[3] % 2 == 1 and tok[4] in (5, 1000) and tok[7] < 3
    _, lp = S.sample_given(x.to(dev), u.to(dev), want_logprob=True)
    assert lp[0] == lp[1] == -math.inf and lp[2] == 0


@pytest.mark.parametrize("dev", DEVICES)
def test_ends_of_the_unit_interval(dev):
    """u = 0 takes the first kept token, the largest u below 1 (and anything beyond) the last."""
    x = logits(4, 700, 1)
    u = torch.tensor([0.0, 1 - 2.0 ** -53, 1.0, 7.0], dtype=torch.float64)
    tok, _ = S.sample_given(x.to(dev), u.to(dev), torch.ones(4, device=dev))
    assert tok.tolist() == [0, 699, 699, 699]
    tok = run(x[:2], u[:2], 1.0, 30, 1.0, 0.0, dev)
    order = [sorted(sorted(range(700), key=lambda i: (-float(x[b, i]), i))[:30]) for b in range(2)]
    assert tok.tolist() == [order[0][0], order[1][-1]]


@pytest.mark.parametrize("dev", DEVICES)
def test_pitch_alignment_and_out(dev):
    """Rows that begin at any element, wider pitches, a given destination."""
    room = torch.randn((5, 4100), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    u = uniform(5, 2).to(dev)
    t = torch.ones(5, device=dev)
    k = torch.full((5,), 40, dtype=torch.int32, device=dev)
    for a, b in ((0, 4096), (3, 4000), (1, 4100)):
        x = room[:, a:b]
        out = torch.full((5,), -1, dtype=torch.int64, device=dev)
        got, _ = S.sample_given(x, u, t, k, out=out)
        want, _ = S.sample_given(x.contiguous(), u, t, k)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
        assert want.tolist() == [R.token(r, v, 1.0, 40, 1.0, 0.0) for r, v in zip(x.cpu().double().tolist(), u.cpu().tolist())]


@pytest.mark.parametrize("dev", DEVICES)
def test_settings_that_are_no_numbers(dev):
    """A temperature that is NaN is greedy, any other setting that is NaN is off, a number that is NaN draws as 0; an infinite temperature is flat."""
    x, u = logits(5, 900, 2), uniform(5, 3)
    x[4, 100:] = -math.inf
    nan = math.nan
    run(x, u, [nan, 1.0, 1.0, 1.0, math.inf], [0, 20, 0, 0, 500], [0.9, nan, 0.9, 1.0, 1.0], [0.0, 0.0, nan, nan, 0.0], dev)
    v = u.clone()
    v[1] = nan
    t = torch.ones(5, device=dev)
    a, _ = S.sample_given(x.to(dev), v.to(dev), t)
    b, _ = S.sample_given(x.to(dev), v.nan_to_num(0.0).to(dev), t)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
def test_cuts_that_need_more_than_the_list(dev):
    """Logits in groups of many equal ones, at every distance: cuts inside a group, top-k and top-p in different groups, long lists and short ones."""
    V, g = 18000, torch.Generator().manual_seed(1)
    levels = torch.tensor([3.0, 2.99, 2.5, 2.0, 0.0, -1.0, -9.0, -40.0])
    x = levels[torch.multinomial(torch.tensor([0.002, 0.01, 0.05, 0.3, 0.3, 0.2, 0.1, 0.038]), V, replacement=True, generator=g)].expand(12, V).clone()
    k = [0, 0, 0, 100, 1500, 7000, 9000, 17900, 3000, 12000, 30, 5]
    p = [0.5, 0.9, 0.999, 1.0, 1.0, 1.0, 0.7, 0.5, 0.9, 0.3, 0.2, 0.999]
    for dtype in (torch.float32, torch.float16):
        for t in (1.0, 0.3, 4.0):
            run(x.to(dtype), uniform(12, 7), t, k, p, [0.0, 0.0, 0.02] * 4, dev)


@pytest.mark.gpu
def test_streams_and_graphs():
    """On a stream of its own, and captured: replays follow what the buffers hold."""
    x, u = logits(6, 5000, 5).cuda(), uniform(6, 6).cuda()
    t, k, p = torch.ones(6, device="cuda"), torch.full((6,), 300, dtype=torch.int32, device="cuda"), torch.full((6,), 0.9, device="cuda")
    want = [S.sample_given(y, u, t, k, p)[0].tolist() for y in (x, x.flip(0))]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a, _ = S.sample_given(x, u, t, k, p)
    s.synchronize()
    assert a.tolist() == want[0]
    y = x.clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o, _ = S.sample_given(y, u, t, k, p)
        graphs.append((gr, o))
    y.copy_(x.flip(0))
    for gr, _ in graphs:
        gr.replay()
    torch.cuda.synchronize()
    assert [o.tolist() for _, o in graphs] == [want[1]] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("V", [131072, 262144])
def test_long_rows(V):
    """Vocabularies that one pass over shared memory does not hold, up to the longest."""
    run(logits(3, V, 1), uniform(3, 2), 1.0, [0, 0, 3000], [1.0, 0.95, 0.9], 0.0, "cuda", check_lp=False)
    run(torch.zeros((2, V)), uniform(2, 2), 1.0, [V - 1, 0], [1.0, 0.5], 0.0, "cuda", check_lp=False)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [9000, 20001, 40000, 70001])
def test_rows_alone_and_in_batches(dev, V):
    """A row's token is the same whatever stands beside it, however many CTAs a row of so many has: every kind of row alone and among 17, 40 and 70."""
    x = logits(10, V, V, 1.5, torch.float32)
    x[3] = 0.25                                                        # equal logits
    x[4] = 1 + x[4] * 1e-4                                             # a narrow range
    x[5, ::2], x[6] = -math.inf, -math.inf
    x[7, V - 3] = math.inf
    x[8, 5:V - 5] = math.nan
    t = [1.0, 0.7, 1.3, 1.0, 1.0, 1.0, 1.0, 1.0, 2.0, 0.0]
    k = [0, 50, V // 2, 0, V - 9, 0, 0, 0, 7, 0]
    p = [0.95, 0.9, 0.8, 0.6, 1.0, 1.0, 0.9, 0.9, 1.0, 1.0]
    m = [0.0, 0.0, 0.001, 0.0, 0.0, 0.01, 0.0, 0.0, 0.0, 0.0]
    u = uniform(10, 3)
    want = [R.token(x[b].nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).double().tolist(), float(u[b]), t[b], k[b], p[b], m[b]) for b in range(10)]
    to = lambda a, dt: torch.tensor(a, dtype=dt, device=dev)
    args = (x.to(dev), u.to(dev), to(t, torch.float32), to(k, torch.int32), to(p, torch.float32), to(m, torch.float32))
    alone = [S.sample_given(*(a[b:b + 1] for a in args), want_logprob=True) for b in range(10)]
    assert [int(o) for o, _ in alone] == want
    lp = torch.cat([q for _, q in alone])
    for B in (17, 40, 70):
        at = torch.arange(B, device=dev) % 10
        tok, q = S.sample_given(*(a[at] for a in args), want_logprob=True)
        assert tok.tolist() == [want[b % 10] for b in range(B)]
        # the sums differ by the order of additions in 64 bits: by a rounding of the 32-bit logarithm (up to 12) and of a difference of it (up to 32)
        assert torch.allclose(q, lp[at], rtol=0.0, atol=2.0 ** -20, equal_nan=True)


@pytest.mark.gpu
def test_long_rows_captured_side_by_side():
    """Two captured calls over rows of several CTAs, replayed on two streams at once, follow what their buffers hold."""
    xs, u = [logits(4, 70001, s).cuda() for s in range(4)], uniform(4, 6).cuda()
    t, k, p = torch.ones(4, device="cuda"), torch.tensor([0, 300, 0, 9], dtype=torch.int32, device="cuda"), torch.full((4,), 0.9, device="cuda")
    want = [S.sample_given(x, u, t, k, p)[0].tolist() for x in xs]
    assert want[0] == [R.token(xs[0][b].double().tolist(), float(u[b]), 1.0, int(k[b]), float(p[b]), 0.0) for b in range(4)]
    held = [xs[0].clone(), xs[1].clone()]
    torch.cuda.synchronize()
    graphs = []
    for y in held:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o, _ = S.sample_given(y, u, t, k, p)
        graphs.append((gr, o))
    held[0].copy_(xs[2])
    held[1].copy_(xs[3])
    torch.cuda.synchronize()
    for s, (gr, _) in zip((torch.cuda.Stream(), torch.cuda.Stream()), graphs):
        with torch.cuda.stream(s):
            for _ in range(20):
                gr.replay()
    torch.cuda.synchronize()
    assert [o.tolist() for _, o in graphs] == want[2:]


def test_refusals():
    x, u = torch.zeros((3, 10)), torch.zeros(3, dtype=torch.float64)
    for kw in (dict(u=u.float()), dict(u=u[:2]), dict(temperature=torch.ones(3, dtype=torch.float64)), dict(temperature=torch.ones(2)),
               dict(top_k=torch.ones(3)), dict(top_p=torch.ones(1)), dict(min_p=torch.ones(3, dtype=torch.bfloat16)), dict(out=torch.zeros(3)),
               dict(out=torch.zeros(4, dtype=torch.int64)), dict(logits=torch.zeros((3, 0))), dict(logits=torch.zeros((3, (1 << 18) + 1)))):
        with pytest.raises(ValueError):
            S.sample_given(**(dict(logits=x, u=u) | kw))
