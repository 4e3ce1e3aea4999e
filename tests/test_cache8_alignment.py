"""Pages, rotation tables and accumulators that begin where no vector access of the 8-bit cache's kernels may: refused on the host, before any launch.

Everything here runs on the host: tensors that say they are on a GPU, and a stand-in for the library that only notes that it was reached."""
import pytest
import torch

from dlti_b200.ops import _lib, kv8
from dlti_b200.ops.elementwise import rope_tables

HD, H, KV, BS = 128, 4, 2, 16


class Elsewhere(torch.Tensor):
    is_cuda = True


def at(t, off):
    """t's numbers in storage that begins `off` bytes behind a multiple of 64."""
    n = t.numel() * t.element_size()
    room = torch.zeros(n + 192, dtype=torch.uint8)
    room = room[-room.data_ptr() % 64 + off:][:n].view(t.dtype).view(t.shape)
    assert room.data_ptr() % 64 == off
    return torch.Tensor._make_subclass(Elsewhere, room.copy_(t))


@pytest.fixture
def reached(monkeypatch):
    calls = []
    monkeypatch.setattr(kv8, "_check_device", lambda op, *t: 0)
    monkeypatch.setattr(kv8, "_stream", lambda d: 0)
    monkeypatch.setattr(kv8, "_bound", {n: (lambda *a, n=n: calls.append(n) or 0) for n in kv8._SIGNATURES})
    return calls


def tensors():
    cos, sin = rope_tables(8, HD, 10000.0, "cpu")
    page = torch.zeros((4, KV, BS, HD), dtype=torch.uint8).view(torch.float8_e4m3fn)
    t = dict(x=torch.zeros((3, (H + 2 * KV) * HD), dtype=torch.bfloat16), acc=torch.zeros((3, (H + 2 * KV) * HD)), cos=cos, sin=sin, k8=page, v8=page,
             ks=torch.ones(4, KV), vs=torch.ones(4, KV), pos=torch.zeros(3, dtype=torch.int32), slots=torch.tensor([0, 1, -1]),
             tables=torch.zeros((3, 2), dtype=torch.int32), ctx=torch.ones(3, dtype=torch.int32))
    return {n: at(a, 0) for n, a in t.items()}


CALLS = {
    "rope_cache8": lambda t: kv8.rope_cache8_(t["x"], t["pos"], t["cos"], t["sin"], t["slots"], t["k8"], t["v8"], t["ks"], t["vs"], H, KV, HD),
    "acc_rope_cache8": lambda t: kv8.acc_rope_cache8(t["acc"], torch.bfloat16, t["pos"], t["cos"], t["sin"], t["slots"], t["k8"], t["v8"], t["ks"], t["vs"],
                                                     H, KV, HD),
    "paged_decode8": lambda t: kv8.paged_decode8(t["x"], t["k8"], t["v8"], t["ks"], t["vs"], t["tables"], t["ctx"], H, KV, HD),
    "gather_rows8": lambda t: kv8.gather_rows8_(t["x"], t["slots"][:2], t["slots"][:2], t["k8"], t["v8"], t["ks"], t["vs"], H, KV, HD),
}


@pytest.mark.parametrize("op,name,offs", [
    ("rope_cache8", "k8", (1, 4, 8)), ("rope_cache8", "v8", (1, 4, 8)), ("rope_cache8", "cos", (4, 8)), ("rope_cache8", "sin", (4, 8)), ("rope_cache8", "x", (2, 8)),
    ("acc_rope_cache8", "k8", (1, 8)), ("acc_rope_cache8", "v8", (8,)), ("acc_rope_cache8", "cos", (4,)), ("acc_rope_cache8", "sin", (8,)),
    ("acc_rope_cache8", "acc", (4, 8)),
    ("paged_decode8", "k8", (1, 4, 8)), ("paged_decode8", "v8", (1, 4, 8)), ("paged_decode8", "x", (2, 8)),
    ("gather_rows8", "k8", (1, 4)), ("gather_rows8", "v8", (1, 4)), ("gather_rows8", "x", (8,))])      # it reads pieces of 8 bytes
def test_refused(reached, op, name, offs):
    for off in offs:
        t = tensors()
        t[name] = at(t[name], off)
        with pytest.raises(ValueError, match=op if name not in ("cos", "sin") else "rotation tables"):
            CALLS[op](t)
    assert not reached


@pytest.mark.parametrize("op", CALLS)
def test_taken(reached, op):
    """The smallest alignments that suffice, and scales anywhere."""
    for off in (0, 16):
        t = {n: at(a, off) for n, a in tensors().items()}
        t["ks"], t["vs"] = at(t["ks"], 4), at(t["vs"], 12)
        CALLS[op](t)
    if op == "gather_rows8":
        t["k8"], t["v8"] = at(t["k8"], 8), at(t["v8"], 8)
        CALLS[op](t)
    assert set(reached) == {"dlti_" + op} and len(reached) == (3 if op == "gather_rows8" else 2)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that nobody may read")
def test_c_entries():
    """The same at the C entries, which refuse before they launch."""
    A = 4096                                                             # addresses that nobody reads
    fn = lambda name: _lib.fn(name, list(kv8._SIGNATURES[name]))
    want = [("dlti_rope_cache8", [A, 8 * HD, A, 8 * HD, A, A, A, A, A, A, A, A, 3, H, KV, HD, BS, 0, None], (0, 2, 5, 6, 8, 9), (1, 3)),
            ("dlti_acc_rope_cache8", [A, A, 8 * HD, A, A, A, A, A, A, A, A, 3, H, KV, HD, BS, 0, None], (0, 1, 4, 5, 7, 8), (2,)),
            ("dlti_paged_decode8", [A, 8 * HD, A, A, A, A, A, 2, A, 3, BS, H, KV, HD, 0.1, 1, None, A, 4 * HD, 0, None], (0, 2, 3), (1,)),
            ("dlti_gather_rows8", [A, 8 * HD, A, A, A, A, A, A, 3, H, KV, HD, BS, 0, None], (0,), (1,))]
    for name, args, pointers, pitches in want:
        for i, more in [(i, 8) for i in pointers] + [(i, 4) for i in pitches]:
            a = list(args)
            a[i] += more
            assert fn(name)(*a) == -1, (name, i)
            assert b"16 bytes" in _lib.gpu_lib().dlti_last_error()
    for i in (4, 5):
        a = list(want[3][1])
        a[i] += 4
        assert fn("dlti_gather_rows8")(*a) == -1 and b"8 bytes" in _lib.gpu_lib().dlti_last_error()
