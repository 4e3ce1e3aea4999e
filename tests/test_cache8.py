"""The 8-bit cache of keys and values against its rules in double precision (tests/ref_cache8.py): restatements on the CPU, kernels on the GPU."""
import math

import pytest
import torch

from dlti_b200.ops import _debug, _lib, kv8
from dlti_b200.ops import serving as S
from dlti_b200.ops.elementwise import rope_tables
from . import ref_cache8 as R

HD = 128
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
E4 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


def pages(n, KV, bs, seed, spread=0.0, dev="cpu"):
    """Pages whose scales differ by up to 2^+-spread; every byte holds a number."""
    g = gen(seed)
    x = torch.randn((n, KV, bs, HD), generator=g)
    x = x * torch.exp2(torch.round((torch.rand((n, KV, 1, 1), generator=g) * 2 - 1) * spread))
    s = kv8.scale_for(x.abs().amax((2, 3)))
    return (x / s[..., None, None]).to(E4).to(dev), s.to(dev)


def table_of(counts, n, seed):
    """Shuffled pages for sequences with `counts` pages each; entries behind a sequence's pages name page 0."""
    perm = torch.randperm(n, generator=gen(seed)).tolist()
    t = torch.zeros((len(counts), max(max(counts), 1)), dtype=torch.int32)
    for i, c in enumerate(counts):
        t[i, :c] = torch.tensor([perm.pop() for _ in range(c)], dtype=torch.int32)
    return t


# ---- rows ---------------------------------------------------------------------------------------------------------------------
def rows_case(seqs, H, KV, bs, dtype, dev, seed=0, pad=0, edit=None, acc=False, apart=False):
    """seqs: (tokens in the cache, tokens that come) of each sequence. Runs the op and the rules, compares everything."""
    g = gen(seed)
    width = (H + 2 * KV) * HD
    T = sum(n for _, n in seqs) + pad
    x = torch.randn((T, width), generator=g).to(dtype)
    counts = [-(-(a + n) // bs) for a, n in seqs]
    P = sum(counts) + 2
    tables = table_of(counts, P, seed + 1)
    slots, pos = [], []
    for i, (a, n) in enumerate(seqs):
        slots += [int(tables[i, j // bs]) * bs + j % bs for j in range(a, a + n)]
        pos += list(range(a, a + n))
    slots, pos = torch.tensor(slots + [-1] * pad), torch.tensor(pos + [0] * pad, dtype=torch.int32)
    k8, ks = pages(P, KV, bs, seed + 2, 3)
    v8, vs = pages(P, KV, bs, seed + 3, 3)
    if edit is not None:
        edit(x, slots, k8, v8, ks, vs)
    cos, sin = rope_tables(max(int(pos.max()) + 1, 2), HD, 10000.0, "cpu")
    cos, sin = cos.contiguous(), sin.contiguous()
    to = lambda t: t.to(dev).clone()
    dk, dv, dks, dvs = to(k8), to(v8), to(ks), to(vs)
    args = (to(pos), to(cos), to(sin), to(slots), dk, dv, dks, dvs, H, KV, HD)
    if acc:
        a = to(x.float())
        got = kv8.acc_rope_cache8(a, dtype, *args)
        assert int((a != 0).sum()) == 0
    elif apart:
        a = to(x)
        got = kv8.rope_cache8_(a, *args, out=torch.full_like(a, 7.0))
        assert torch.equal(a.cpu().view(torch.int16), x.view(torch.int16))
    else:
        a = to(x)
        got = kv8.rope_cache8_(a, *args)
        assert got.data_ptr() == a.data_ptr()
    got = got.cpu()
    want = R.rotate(x.double(), pos.long(), cos.to(dtype).double(), sin.to(dtype).double(), H + KV, HD)
    fin = torch.isfinite(want)
    # one rounding to the type (half a step, or half of the finest one) after one in fp32 of numbers of the size of both terms
    size = torch.zeros_like(want)
    xa = x.double().abs().view(T, -1, 2, HD // 2)
    size.view(T, -1, 2, HD // 2)[:] = xa.sum(2, keepdim=True)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -23 * size + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    turned = torch.arange(want.shape[1]) < (H + KV) * HD      # values are not touched: compared bit by bit below
    assert bool(((got.double() - want).abs() <= tol)[fin & turned].all())
    assert torch.equal(got[:, (H + KV) * HD:].contiguous().view(torch.int16), x[:, (H + KV) * HD:].contiguous().view(torch.int16))
    # the cache takes the rows as they left, and rounds once
    ok = slots >= 0
    kv = got[ok][:, H * HD:].reshape(-1, 2, KV, HD).double()
    for new, q, s, dq, ds in ((kv[:, 0], k8, ks, dk, dks), (kv[:, 1], v8, vs, dv, dvs)):
        rq, rs = q.double(), s.double()
        R.write(new, slots[ok], rq, rs)
        assert torch.equal(ds.cpu().double(), rs)
        d = dq.cpu().double()
        assert bool(((d == rq) | (d.isnan() & rq.isnan())).all())
    return got, (dk, dv, dks, dvs)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seqs,H,KV,bs,pad", [
    ([(0, 1)], 1, 1, 8, 0),                                  # one row, one head, a page of its own
    ([(5, 1), (16, 1), (31, 1), (700, 1)], 8, 2, 16, 3),     # decode rows: inside a page, at its begin, at its end
    ([(0, 37), (13, 40), (16, 16), (47, 1)], 6, 3, 16, 0),   # portions that begin inside pages
    ([(3, 70), (0, 33)], 5, 5, 32, 2),                       # more rows of a page than a warp keeps in registers
    ([(60, 100)], 16, 1, 64, 0),
    ([(0, 30), (9, 31)], 4, 4, 24, 0),                       # pages that are no power of two
    ([(8, 1)] * 70, 9, 1, 8, 0),                             # query heads that do not fill a warp's share
])
def test_rows(dev, dtype, seqs, H, KV, bs, pad):
    got, cache = rows_case(seqs, H, KV, bs, dtype, dev, seed=len(seqs) + bs, pad=pad)
    again, other = rows_case(seqs, H, KV, bs, dtype, dev, seed=len(seqs) + bs, pad=pad, apart=True)
    from_acc, third = rows_case(seqs, H, KV, bs, dtype, dev, seed=len(seqs) + bs, pad=pad, acc=True)
    assert torch.equal(got, again) and torch.equal(got, from_acc)
    for a, b, c in zip(cache, other, third):
        a, b, c = (t.view(torch.uint8) if t.dtype == E4 else t for t in (a, b, c))
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_of_many_pages(dev):
    """Enough rows that a warp serves sixteen of them: pages begin anywhere in these sixteen, and go on in the next."""
    rows_case([(5, 400), (0, 301), (11, 5), (16, 3), (7, 90)], 8, 8, 16, torch.bfloat16, dev, seed=4)
    rows_case([(5, 400), (0, 301), (11, 5), (40, 3), (7, 90)], 16, 8, 32, torch.float16, dev, seed=5)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_raise_and_keep_scales(dev, dtype):
    """A larger row raises its page's scale by 2^1 .. 2^30 and what is there is rounded; a smaller one does not touch it. Zeros, too."""
    def edit(x, slots, k8, v8, ks, vs):
        big = 60000.0 if dtype == torch.float16 else 2.0 ** 30
        x[0] *= 100
        x[1] *= big / 8
        x[2] *= 1e-4
        x[3] = 0
        x[4] *= 1e-6
    rows_case([(5, 1), (3, 1), (9, 1), (2, 1), (0, 1)], 4, 2, 16, dtype, dev, seed=9, edit=edit)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_infinities_and_nan(dev, dtype):
    """Values (which are not rotated): infinities take the largest number of their page and do not raise it, NaN stays; a page that begins anew does
    not look at the numbers or the scale left in it."""
    H, KV, bs = 2, 2, 16
    def edit(x, slots, k8, v8, ks, vs):
        v = x[:, (H + KV) * HD:]
        v[0, 3], v[0, 4], v[1, 130], v[2, 7] = math.inf, -math.inf, math.nan, math.inf
        v[3] = math.inf
        v[4, :] = math.nan
        first = int(slots[5]) // bs
        v8.view(torch.uint8)[first] = 0x7f                   # NaN everywhere
        vs[first] = 2.0 ** 100
    _, (k8, v8, ks, vs) = rows_case([(5, 2), (7, 1), (9, 1), (4, 1), (0, 3)], H, KV, bs, dtype, dev, seed=3, edit=edit)
    assert float(vs.max()) < 2.0 ** 10


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_extreme_numbers(dev):
    """bf16 at both ends of its range: scales stop at 2^-120 and 2^120."""
    def edit(x, slots, k8, v8, ks, vs):
        x[0, :], x[1, :], x[2, :] = 2.0 ** -130, 3.3e38, 448.0 * 2.0 ** -20
        x[0, 5], x[3, :] = -(2.0 ** -133), 0.0
        x[:, :4 * HD] = 0                                    # queries and keys: a rotation would leave the range
    _, (_, _, _, vs) = rows_case([(0, 1)] * 4, 2, 2, 16, torch.bfloat16, dev, seed=6, edit=edit)
    assert {float(s) for s in vs.unique()} >= {2.0 ** -120, 2.0 ** 120, 2.0 ** -20}


@pytest.mark.parametrize("dev", DEVICES)
def test_page_written_row_by_row(dev):
    """A page that fills one row a step: each number as if written with the scale it got, rounded again whenever the scale rose."""
    KV, bs, dtype = 2, 16, torch.bfloat16
    g = gen(5)
    k8, ks = pages(3, KV, bs, 1, 2, dev)
    v8, vs = pages(3, KV, bs, 2, 2, dev)
    rq, rs = v8.cpu().double(), vs.cpu().double()
    cos, sin = rope_tables(64, HD, 10000.0, dev)
    for j in range(bs):
        x = (torch.randn((1, 4 * KV * HD), generator=g) * 2.0 ** (j % 7)).to(dtype)
        slots = torch.tensor([bs + j])
        kv8.rope_cache8_(x.to(dev).clone(), torch.tensor([j], dtype=torch.int32, device=dev), cos, sin, slots.to(dev), k8, v8, ks, vs, 2 * KV, KV, HD)
        R.write(x[:, 3 * KV * HD:].view(1, KV, HD).double(), slots, rq, rs)
    assert torch.equal(v8.cpu().double(), rq) and torch.equal(vs.cpu().double(), rs)


# ---- attention ----------------------------------------------------------------------------------------------------------------
def attend_case(lens, H, KV, bs, dtype, dev, seed=0, spread=3.0, scale=None, max_ctx=None, edit=None, wide=0, q_gain=1.0):
    g = gen(seed)
    counts = [-(-n // bs) for n in lens]
    P = sum(counts) + 2
    table = table_of(counts, P, seed + 1)
    if wide:
        table = torch.cat([table, torch.zeros((len(lens), wide), dtype=torch.int32)], 1)
    k8, ks = pages(P, KV, bs, seed + 2, spread)
    v8, vs = pages(P, KV, bs, seed + 3, spread)
    ctx = torch.tensor(lens, dtype=torch.int32)
    for i, n in enumerate(lens):                             # what a page holds behind the end is no number
        if n % bs:
            k8.view(torch.uint8)[int(table[i, n // bs]), :, n % bs:] = 0x7f
            v8.view(torch.uint8)[int(table[i, n // bs]), :, n % bs:] = 0xff
    buf = (torch.randn((len(lens), (H + 2 * KV) * HD), generator=g) * q_gain).to(dtype)
    if edit is not None:
        edit(buf, k8, v8, ks, vs, table)
    sc = scale if scale is not None else 1.0 / math.sqrt(HD)
    to = lambda t: t.to(dev)
    got = kv8.paged_decode8(to(buf), to(k8), to(v8), to(ks), to(vs), to(table), to(ctx), H, KV, HD, scale, max_ctx=max_ctx).cpu()
    out, mag, reach = R.attend(buf, k8, v8, ks, vs, table, ctx, H, KV, HD, sc)
    return got, out, R.attend_error(out, mag, reach, ctx, dtype, HD)


def check_attend(*a, **kw):
    got, want, tol = attend_case(*a, **kw)
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,H,KV,bs", [
    ([1], 1, 1, 16), ([0, 0], 2, 1, 16), ([7, 8, 9, 15, 16, 17, 0, 1, 31, 33], 4, 2, 16),
    ([7, 8, 9, 23, 24, 25, 100], 3, 1, 8), ([47, 48, 49, 200], 10, 2, 24), ([63, 64, 65, 130], 8, 1, 64),
    ([300, 1000, 511, 3], 16, 2, 16), ([129, 77], 18, 2, 16), ([100, 400], 16, 1, 32), ([90, 5], 17, 1, 16), ([64, 2000], 32, 32, 16),
])
def test_attend(dev, dtype, lens, H, KV, bs):
    check_attend(lens, H, KV, bs, dtype, dev, seed=len(lens) + H)


def test_splits_are_clusters_of_one_size():
    for ctas in (*range(1, 500), 5000):
        for reach in (1, 64, 65, 600, 5000, 100000):
            n = kv8.splits8(ctas, reach)
            assert 1 <= n <= 128 and n % -(-n // 8) == 0 and n <= max(1, -(-reach // 64)) and (n == 1 or n * ctas <= 444)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("max_ctx", [None, 100, 4096])
def test_attend_reach(dev, max_ctx):
    """A table wider than the contexts, and a given reach that is smaller or larger than they are: the same answer."""
    check_attend([257, 90, 0, 1500], 8, 2, 16, torch.bfloat16, dev, seed=2, max_ctx=max_ctx, wide=40)


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_context_behind_the_table(dev):
    """A length that the table does not hold ends with the table."""
    k8, ks = pages(6, 1, 16, 1, 1, dev)
    v8, vs = pages(6, 1, 16, 2, 1, dev)
    q = torch.randn((1, 2 * HD), generator=gen(1)).to(torch.bfloat16).to(dev)
    t = torch.tensor([[3, 1]], dtype=torch.int32, device=dev)
    a, b = (kv8.paged_decode8(q, k8, v8, ks, vs, t, torch.tensor([n], dtype=torch.int32, device=dev), 2, 1, HD) for n in (32, 1000))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("spread", [12.0, 30.0])
def test_attend_pages_of_very_different_size(dev, spread):
    """Scales from page to page by factors of 2^+-12 and 2^+-30 (bf16: values of that size do not fit fp16)."""
    check_attend([40, 300, 17], 4, 2, 16, torch.bfloat16, dev, seed=8, spread=spread, scale=2.0 ** -spread * 0.05)


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_weight_on_the_page_of_small_values(dev):
    """All weight on tokens whose values are 2^-20 of the largest in the context: they keep their bits."""
    def edit(q, k8, v8, ks, vs, table):
        ks[table[0, 0].long()] *= 64
        vs[table[0, 1:4].long()] *= 2.0 ** 20
    check_attend([64], 4, 1, 16, torch.bfloat16, dev, seed=3, spread=0.0, edit=edit, q_gain=4.0, scale=0.3)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_scores_that_stand_out(dev, dtype):
    """Sharp softmax: scores of hundreds, of either sign, the largest anywhere; a scale of zero averages; a negative one is a scale, too."""
    for scale in (2.0, -0.5, 0.0):
        check_attend([200, 64, 33], 4, 4, 16, dtype, dev, seed=5, scale=scale, spread=1.0)


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_queries_of_any_size(dev):
    for gain in (2.0 ** -60, 2.0 ** 60):
        check_attend([50, 20], 2, 1, 16, torch.bfloat16, dev, seed=6, q_gain=gain, scale=0.05 / gain)
    def zero(q, *_):
        q[:, :HD] = 0
    check_attend([50, 20], 2, 1, 16, torch.float16, dev, seed=7, edit=zero)
    def small(q, *_):
        q[:, 1:HD] *= 2.0 ** -12                              # fp16 numbers with few bits left
    check_attend([50, 20], 2, 1, 16, torch.float16, dev, seed=8, edit=small)


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_nan_stays_where_it_is(dev):
    """A key that is no number spoils its key head's query heads and no others; a value that is none, its dimension."""
    def edit(q, k8, v8, ks, vs, table):
        k8.view(torch.uint8)[int(table[0, 1]), 0, 3, 9] = 0x7f
        v8.view(torch.uint8)[int(table[1, 0]), 1, 2, 77] = 0x7f
    got, want, tol = attend_case([40, 40, 40], 4, 2, 16, torch.bfloat16, dev, seed=4, edit=edit)
    assert torch.equal(got.isnan(), want.isnan())
    assert bool(got[0, :2 * HD].isnan().all()) and int(got[1].isnan().sum()) == 2 and not bool(got[2].isnan().any())
    ok = ~want.isnan()
    assert bool(((got.double() - want).abs() <= tol)[ok].all())


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_strides_and_out(dev):
    k8, ks = pages(9, 2, 16, 1, 1, dev)
    v8, vs = pages(9, 2, 16, 2, 1, dev)
    t = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    n = torch.tensor([50, 64], dtype=torch.int32, device=dev)
    q = torch.randn((2, 4 * HD), generator=gen(1)).to(torch.float16).to(dev)
    want = kv8.paged_decode8(q, k8, v8, ks, vs, t, n, 4, 2, HD)
    wide = torch.zeros((2, 9 * HD), dtype=torch.float16, device=dev)
    wide[:, :4 * HD] = q
    room = torch.full((2, 6 * HD), 5.0, dtype=torch.float16, device=dev)
    got = kv8.paged_decode8(wide, k8, v8, ks, vs, t, n, 4, 2, HD, out=room[:, HD:5 * HD])
    assert torch.equal(got, want) and torch.equal(room[:, HD:5 * HD], want)
    assert bool((room[:, :HD] == 5).all()) and bool((room[:, 5 * HD:] == 5).all())


# ---- rows read back -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,H,KV,bs", [(1, 1, 1, 8), (37, 6, 3, 16), (300, 8, 1, 24), (0, 2, 2, 16)])
def test_gather(dev, dtype, n, H, KV, bs):
    P = n // bs + 3
    k8, ks = pages(P, KV, bs, 1, 4)
    v8, vs = pages(P, KV, bs, 2, 4)
    slots = torch.randperm(P * bs, generator=gen(3))[:n]
    rows = torch.randperm(n + 5, generator=gen(4))[:n]
    ext = torch.randn((n + 5, (H + 2 * KV) * HD), generator=gen(5)).to(dtype)
    want = ext.clone()
    for i in range(n):
        p, o = int(slots[i]) // bs, int(slots[i]) % bs
        want[rows[i], H * HD:(H + KV) * HD] = (k8[p, :, o].double() * ks[p][:, None].double()).flatten().to(dtype)
        want[rows[i], (H + KV) * HD:] = (v8[p, :, o].double() * vs[p][:, None].double()).flatten().to(dtype)
    to = lambda t: t.to(dev)
    e = to(ext).clone()
    got = kv8.gather_rows8_(e, to(rows), to(slots), to(k8), to(v8), to(ks), to(vs), H, KV, HD)
    assert got.data_ptr() == e.data_ptr() and torch.equal(got.cpu(), want)


# ---- as programs call them ----------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_far_pages():
    """Caches of more than 2^31 bytes: rows written to their last pages, read back and attended to, as near the begin of a small one."""
    n, KV, bs = (1 << 20) + 700, 1, 16
    far = [n - 1, n - 300, n - 2, (1 << 20) + 1, 5]
    big = [torch.zeros((n, KV, bs, HD), dtype=torch.uint8, device="cuda").view(E4) for _ in range(2)]
    small = [torch.zeros((5, KV, bs, HD), dtype=torch.uint8, device="cuda").view(E4) for _ in range(2)]
    cos, sin = rope_tables(80, HD, 10000.0, "cuda")
    x = torch.randn((70, 4 * HD), generator=gen(1)).to(torch.bfloat16).cuda()
    got = []
    for (k, v), pages_ in ((big, far), (small, [0, 1, 2, 3, 4])):
        ks, vs = (torch.full(k.shape[:2], 2.0 ** -120, device="cuda") for _ in range(2))
        slots = torch.tensor([pages_[j // bs] * bs + j % bs for j in range(70)], device="cuda")
        rows = kv8.rope_cache8_(x.clone(), torch.arange(70, dtype=torch.int32, device="cuda"), cos, sin, slots, k, v, ks, vs, 2, KV, HD)
        ext = torch.zeros_like(rows)
        kv8.gather_rows8_(ext, torch.arange(70, device="cuda"), slots, k, v, ks, vs, 2, KV, HD)
        t = torch.tensor([pages_], dtype=torch.int32, device="cuda")
        o = kv8.paged_decode8(rows[-1:], k, v, ks, vs, t, torch.tensor([70], dtype=torch.int32, device="cuda"), 2, KV, HD)
        got.append((rows, ext, o))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and float(got[0][2].abs().sum()) > 0


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bs", [8, 16, 24])
def test_table_entries_behind_the_context(dev, bs):
    """They are not read: any number may stand there."""
    def edit(q, k8, v8, ks, vs, table):
        for i, n in enumerate((3 * bs, 2 * bs + 5, 0, 1)):
            table[i, -(-n // bs):] = 1 << 30
    check_attend([3 * bs, 2 * bs + 5, 0, 1], 4, 2, bs, torch.bfloat16, dev, seed=1, edit=edit, wide=9, max_ctx=5000)


@pytest.mark.gpu
@pytest.mark.parametrize("reach", [64, 700, 60000])
def test_streams_and_graphs(reach):
    """A decode step (rows, attention) on a stream of its own, and captured twice: the graphs share nothing but the cache, are replayed side by side
    on two streams, and follow what their buffers hold."""
    KV, H, bs, B = 2, 8, 16, 3
    width = max(4, reach // bs)
    n = 3 * 50 + 1
    cache = (*pages(n, KV, bs, 1, 1, "cuda"), *pages(n, KV, bs, 2, 1, "cuda"))
    k8, ks, v8, vs = cache
    table = torch.zeros((B, width), dtype=torch.int32)
    for b in range(B):
        table[b, :min(width, 50)] = torch.arange(50)[:width] + 50 * b
    table = table.cuda()
    cos, sin = rope_tables(900, HD, 10000.0, "cuda")
    lens = torch.tensor([5, 60, 33], dtype=torch.int32, device="cuda")
    x = torch.randn((B, (H + 2 * KV) * HD), generator=gen(3)).to(torch.bfloat16).cuda()

    slots = torch.tensor([int(table[b, (m - 1) // bs]) * bs + (m - 1) % bs for b, m in enumerate(lens.tolist())], device="cuda")

    def step(x, kk, kss, vv, vss):
        rows = kv8.rope_cache8_(x, lens - 1, cos, sin, slots, kk, vv, kss, vss, H, KV, HD, out=torch.empty_like(x))
        return kv8.paged_decode8(rows, kk, vv, kss, vss, table, lens, H, KV, HD, max_ctx=reach)

    fresh = lambda: tuple(t.clone() for t in cache)
    want = [step(y, *fresh()).clone() for y in (x, x * 2)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    mine = fresh()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = step(x, *mine)
    s.synchronize()
    assert torch.equal(got, want[0])
    sets = []
    for _ in range(2):
        y, c = x.clone(), fresh()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(y, *c)
        sets.append((g, y, o))
    sets[1][1].copy_(x * 2)
    torch.cuda.synchronize()
    for (g, _, _), stream in zip(sets, (s, torch.cuda.Stream())):
        with torch.cuda.stream(stream):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(sets[0][2], want[0]) and torch.equal(sets[1][2], want[1])


# ---- refusals -------------------------------------------------------------------------------------------------------------------
def test_refusals():
    k8, ks = pages(4, 2, 16, 1)
    v8, vs = pages(4, 2, 16, 2)
    x = torch.zeros((3, 8 * HD), dtype=torch.bfloat16)
    pos, slots = torch.zeros(3, dtype=torch.int32), torch.tensor([0, 1, -1])
    cos, sin = rope_tables(8, HD, 10000.0, "cpu")
    t, n = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)

    def rows(**kw):
        a = dict(qkv=x, pos=pos, cos_t=cos, sin_t=sin, slots=slots, k8=k8, v8=v8, k_scale=ks, v_scale=vs, H=4, KV=2, hd=HD) | kw
        return kv8.rope_cache8_(**a)

    def attend(**kw):
        a = dict(q=x, k8=k8, v8=v8, k_scale=ks, v_scale=vs, block_tables=t, ctx_lens=n, H=4, KV=2, hd=HD) | kw
        return kv8.paged_decode8(**a)

    short = pages(4, 2, 4, 1)
    for bad in (dict(KV=1), dict(H=5), dict(hd=64), dict(k8=k8.view(torch.uint8)), dict(k_scale=ks.double()), dict(v_scale=vs[:2]), dict(k8=k8[::2], v8=v8[::2]),
                dict(k8=short[0], v8=short[0], k_scale=short[1], v_scale=short[1])):
        with pytest.raises(ValueError):
            rows(**bad)
        with pytest.raises(ValueError):
            attend(**bad)
        with pytest.raises(ValueError):
            kv8.gather_rows8_(**(dict(ext=x, rows=slots[:2], slots=slots[:2], k8=k8, v8=v8, k_scale=ks, v_scale=vs, H=4, KV=2, hd=HD) | bad))
    for bad in (dict(pos=pos.long()), dict(slots=slots.int()), dict(slots=slots[:2]), dict(out=x.float()), dict(out=x[:2])):
        with pytest.raises(ValueError):
            rows(**bad)
    for bad in (dict(H=3), dict(q=x[:, :HD]), dict(block_tables=t.long()), dict(ctx_lens=n[:2]), dict(out=x.float()), dict(out=x), dict(ctx_lens=n.long())):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(ValueError):
        kv8.acc_rope_cache8(x, torch.bfloat16, pos, cos, sin, slots, k8, v8, ks, vs, 4, 2, HD)
    with pytest.raises(ValueError):
        kv8.gather_rows8_(x, slots[:2], slots, k8, v8, ks, vs, 4, 2, HD)
    assert rows().shape == x.shape and attend().shape == (3, 4 * HD)


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_that_overlap(dev):
    """Rows that are written one over the other are refused; rows that are only read may be one and the same."""
    k8, ks = pages(4, 2, 16, 1, dev=dev)
    v8, vs = pages(4, 2, 16, 2, dev=dev)
    to = lambda a, dt: torch.tensor(a, dtype=dt, device=dev)
    one = torch.ones((1, 8 * HD), dtype=torch.bfloat16, device=dev)
    t, n = torch.zeros((3, 1), dtype=torch.int32, device=dev), to([1, 2, 3], torch.int32)
    o = torch.zeros((1, 4 * HD), dtype=torch.bfloat16, device=dev).expand(3, -1)
    with pytest.raises(ValueError):
        kv8.paged_decode8(one.expand(3, -1), k8, v8, ks, vs, t, n, 4, 2, HD, out=o)
    same = kv8.paged_decode8(one.expand(3, -1), k8, v8, ks, vs, t, n, 4, 2, HD)
    assert torch.equal(same, kv8.paged_decode8(one.repeat(3, 1), k8, v8, ks, vs, t, n, 4, 2, HD))
    cos, sin = rope_tables(8, HD, 10000.0, dev)
    pos, slots = to([0, 1, 2], torch.int32), to([16, 17, 18], torch.int64)
    out = torch.empty((3, 8 * HD), dtype=torch.bfloat16, device=dev)
    if dev == "cuda":
        with pytest.raises(ValueError):
            kv8.rope_cache8_(one.expand(3, -1), pos, cos, sin, slots, k8, v8, ks, vs, 4, 2, HD)
        with pytest.raises(ValueError):
            kv8.rope_cache8_(out, pos, cos, sin, slots, k8, v8, ks, vs, 4, 2, HD, out=one.expand(3, -1))
        with pytest.raises(ValueError):
            kv8.gather_rows8_(one.expand(3, -1), slots - 16, slots, k8, v8, ks, vs, 4, 2, HD)
    kv8.rope_cache8_(one.expand(3, -1), pos, cos, sin, slots, k8, v8, ks, vs, 4, 2, HD, out=out)
    again = one.repeat(3, 1)
    kv8.rope_cache8_(again, pos, cos, sin, slots, k8, v8, ks, vs, 4, 2, HD)
    assert torch.equal(out, again)


@pytest.mark.gpu
def test_tensors_elsewhere():
    """A tensor that is not on the current device is refused, not read."""
    from dlti_b200.ops.pages import copy_pages
    k8, ks = pages(4, 2, 16, 1, dev="cuda")
    v8, vs = pages(4, 2, 16, 2, dev="cuda")
    x = torch.zeros((3, 8 * HD), dtype=torch.bfloat16, device="cuda")
    cos, sin = rope_tables(8, HD, 10000.0, "cuda")
    pos, slots = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([0, 1, -1], device="cuda")
    t, n = torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for i in (1, 2, 3, 4, 5, 6, 7, 8):
        a = [x, pos, cos, sin, slots, k8, v8, ks, vs]
        a[i] = a[i].cpu()
        with pytest.raises(ValueError):
            kv8.rope_cache8_(*a, 4, 2, HD)
    for i in (1, 2, 3, 4, 5, 6):
        a = [x, k8, v8, ks, vs, t, n]
        a[i] = a[i].cpu()
        with pytest.raises(ValueError):
            kv8.paged_decode8(*a, 4, 2, HD)
    with pytest.raises(ValueError):
        kv8.paged_decode8(x, k8, v8, ks, vs, t, n, 4, 2, HD, out=torch.zeros((3, 4 * HD), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        kv8.gather_rows8_(x, slots[:2], slots[:2].cpu(), k8, v8, ks, vs, 4, 2, HD)
    with pytest.raises(ValueError):
        copy_pages([k8, v8.cpu()], [0], [1])
    with pytest.raises(ValueError):
        S.sample_given(x.float(), torch.zeros(3, dtype=torch.float64))
    with pytest.raises(_lib.DltiError):
        kv8.rope_cache8_(torch.zeros((3, 8 * HD), device="cuda"), pos, cos, sin, slots, k8, v8, ks, vs, 4, 2, HD)


def test_index_checks():
    """The opt-in checks name slots outside the cache, slots that occur twice, pages whose rows are apart, tables and lengths that do not fit."""
    k8, ks = pages(4, 1, 16, 1)
    v8, vs = pages(4, 1, 16, 2)
    cos, sin = rope_tables(8, HD, 10000.0, "cpu")
    x = torch.zeros((3, 3 * HD), dtype=torch.bfloat16)
    _debug.enable()
    try:
        for slots in ([0, 64, 1], [3, 3, 4], [0, 17, 1], [5, -1, 6], [-2, 0, 1]):
            with pytest.raises(_debug.DltiIndexError):
                kv8.rope_cache8_(x, torch.zeros(3, dtype=torch.int32), cos, sin, torch.tensor(slots), k8, v8, ks, vs, 1, 1, HD)
        kv8.rope_cache8_(x, torch.zeros(3, dtype=torch.int32), cos, sin, torch.tensor([5, 6, -1]), k8, v8, ks, vs, 1, 1, HD)
        for tables, n in (([[4, 0]], 20), ([[0, -1]], 20), ([[0, 1]], 33)):
            with pytest.raises(_debug.DltiIndexError):
                kv8.paged_decode8(x[:1], k8, v8, ks, vs, torch.tensor(tables, dtype=torch.int32), torch.tensor([n], dtype=torch.int32), 1, 1, HD)
        with pytest.raises(_debug.DltiIndexError):
            kv8.gather_rows8_(x, torch.tensor([5]), torch.tensor([0]), k8, v8, ks, vs, 1, 1, HD)
    finally:
        _debug.enable(False)
