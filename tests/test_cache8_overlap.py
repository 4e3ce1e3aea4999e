"""Destinations that share memory with the rows they are made from: the same rows may be, any other overlap is refused before a launch."""
import pytest
import torch

from dlti_b200.ops import _lib, kv8
from dlti_b200.ops.elementwise import rope_tables
from .test_cache8 import pages

H, KV, HD, BS = 4, 2, 128, 16
W = (H + 2 * KV) * HD
L = 2 * W + 64


def places(w, wide):
    """(first element and pitch of rows of `w` columns that are read, the same of rows of `wide` that are written, their number, whether that is fine)"""
    return [(0, L, 0, L, 3, True),                    # the same rows
            (0, L, W, L, 3, True), (W, L, 0, L, 3, True),      # columns side by side
            (0, L, 3 * L, L, 3, True), (3 * L, L, 0, L, 3, True),      # rows behind
            (0, L, L, L, 3, False), (L, L, 0, L, 3, False),    # a row further
            (0, L, 64, L, 3, False), (64, L, 0, L, 3, False),  # columns that overlap
            (0, L, w - 8, L, 3, False), (0, L, w, L, 3, True), (wide, L, 0, L, 3, True), (wide - 8, L, 0, L, 3, False),
            (0, L, L - 8, L, 3, False), (0, L, 2 * L - wide, L, 3, True),
            (0, L, 0, W, 3, False),                   # other pitches from the same place
            (0, 0, 0, L, 3, False),                   # one row read for all, and written
            (0, L, 0, W, 1, True), (0, L, 64, L, 1, False), (0, L, W, L, 1, True)]      # of one row there is no pitch


def tensors(dev):
    k8, ks = pages(4, KV, BS, 1, dev=dev)
    v8, vs = pages(4, KV, BS, 2, dev=dev)
    room = torch.randn(8 * L, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(dev)
    return k8, v8, ks, vs, room


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that nobody may read")
def test_c_entries():
    """On a machine without a GPU, where a call that is let through ends with CUDA's own error."""
    A, M = 1 << 20, 1 << 30
    for a, la, b, lb, n, ok in places(W, W):
        f = _lib.fn("dlti_rope_cache8", list(kv8._SIGNATURES["dlti_rope_cache8"]))
        rc = f(A + 2 * a, la, A + 2 * b, lb, M, M, M, M, M, M, M, M, n, H, KV, HD, BS, 0, None)
        assert (rc == -1) == (not ok) and rc != 0, (a, la, b, lb, n)
        assert ok or b"overlap" in _lib.gpu_lib().dlti_last_error()
    for a, la, b, lb, n, ok in places(H * HD, H * HD):
        f = _lib.fn("dlti_paged_decode8", list(kv8._SIGNATURES["dlti_paged_decode8"]))
        rc = f(A + 2 * a, la, M, M, M, M, M, 2, M, n, BS, H, KV, HD, 0.1, 1, None, A + 2 * b, lb, 0, None)
        assert (rc == -1) == (not ok) and rc != 0, (a, la, b, lb, n)
        assert ok or b"overlap" in _lib.gpu_lib().dlti_last_error()


@pytest.mark.gpu
def test_rows():
    """Allowed places give what a destination of its own gets; the others raise."""
    cos, sin = rope_tables(8, HD, 10000.0, "cuda")
    for a, la, b, lb, n, ok in places(W, W):
        k8, v8, ks, vs, room = tensors("cuda")
        pos = torch.arange(n, dtype=torch.int32, device="cuda")
        args = (pos, cos, sin, pos.long() + 3, k8, v8, ks, vs, H, KV, HD)
        x, out = room[a:].as_strided((n, W), (la, 1)), room[b:].as_strided((n, W), (lb, 1))
        if not ok:
            with pytest.raises((_lib.DltiError, ValueError)):
                kv8.rope_cache8_(x, *args, out=out)
            continue
        want = kv8.rope_cache8_(x, *args, out=torch.empty((n, W), dtype=x.dtype, device="cuda"))
        assert torch.equal(kv8.rope_cache8_(x, *args, out=out), want)


@pytest.mark.gpu
@pytest.mark.parametrize("max_ctx", [32, 700, 60000])
def test_attention(max_ctx):
    """The same over one split, a cluster and several."""
    for a, la, b, lb, n, ok in places(H * HD, H * HD):
        k8, v8, ks, vs, room = tensors("cuda")
        tables = torch.randint(0, 4, (n, 44), generator=torch.Generator().manual_seed(n), dtype=torch.int32).cuda()
        ctx = torch.tensor([700, 1, 333][:n], dtype=torch.int32, device="cuda")
        args = (k8, v8, ks, vs, tables, ctx, H, KV, HD)
        q, out = room[a:].as_strided((n, H * HD), (la, 1)), room[b:].as_strided((n, H * HD), (lb, 1))
        if not ok:
            with pytest.raises((_lib.DltiError, ValueError)):
                kv8.paged_decode8(q, *args, max_ctx=max_ctx, out=out)
            continue
        want = kv8.paged_decode8(q, *args, max_ctx=max_ctx)
        assert torch.equal(kv8.paged_decode8(q, *args, max_ctx=max_ctx, out=out), want)
