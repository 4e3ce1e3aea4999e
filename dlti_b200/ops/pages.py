"""Copies of cache pages (csrc/pages.cu): what a sequence that goes on from another one's tokens needs of its own."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_P = C.POINTER


def check_copies(src: list[int], dst: list[int], num_pages: int) -> list[tuple[int, int]]:
    """The pairs of a call, without those that copy a page onto itself. Refused: pages outside the cache, a page written twice, a page both read
    and written (copies have no order)."""
    if len(src) != len(dst):
        raise ValueError(f"copy_pages: {len(src)} sources for {len(dst)} destinations")
    if any(not 0 <= p < num_pages for p in (*src, *dst)):
        raise ValueError(f"copy_pages: pages are 0 .. {num_pages - 1}")
    if len(set(dst)) < len(dst):
        raise ValueError("copy_pages: a page is written twice")
    pairs = [(a, b) for a, b in zip(src, dst) if a != b]
    if {a for a, _ in pairs} & {b for _, b in pairs}:
        raise ValueError("copy_pages: a page is both read and written")
    return pairs


def copy_pages(caches: list[torch.Tensor], src: list[int], dst: list[int], page_dim: int = 0) -> None:
    """Pages src[i] -> dst[i] (whole numbers on the host) of every tensor in `caches`: [pages, ...], or with page_dim=1 [layers, pages, ...]. What a
    page holds is contiguous. One launch for up to 32 tensors and 300 pairs."""
    if page_dim not in (0, 1):
        raise ValueError("copy_pages: pages are dimension 0, or dimension 1 behind the layers")
    if not caches:
        return
    counts = {t.shape[page_dim] for t in caches}
    if len(counts) > 1:
        raise ValueError(f"copy_pages: caches of {sorted(counts)} pages")
    pairs = check_copies(src, dst, counts.pop())
    for t in caches:
        one = t.select(page_dim, 0)
        if not (one if page_dim == 0 else one.select(0, 0)).is_contiguous():
            raise ValueError("copy_pages: what a page holds is contiguous")
    if not pairs:
        return
    if not _lib.use_native(*caches):
        a, b = (torch.tensor(p) for p in zip(*pairs))
        for t in caches:
            if page_dim == 0:
                t[b] = t[a]
            else:
                t[:, b] = t[:, a]
        return
    d = torch.cuda.current_device()
    if any(not t.is_cuda or t.device.index != d for t in caches):
        raise ValueError(f"copy_pages: every cache is on the current device, cuda:{d}")
    n = len(caches)
    es = [t.element_size() for t in caches]
    layers = [t.shape[0] if page_dim else 1 for t in caches]
    page = [t.stride(page_dim) * e for t, e in zip(caches, es)]
    layer = [t.stride(0) * e if page_dim else 0 for t, e in zip(caches, es)]
    size = [t[(0,) * (page_dim + 1)].numel() * e for t, e in zip(caches, es)]
    f = _lib.fn("dlti_copy_pages", [C.c_void_p, _P(C.c_int), _P(C.c_longlong), _P(C.c_longlong), _P(C.c_longlong), C.c_int, _P(C.c_int), _P(C.c_int),
                                    C.c_int, C.c_void_p])
    m = len(pairs)
    _lib.check(f((C.c_void_p * n)(*[t.data_ptr() for t in caches]), (C.c_int * n)(*layers), (C.c_longlong * n)(*layer), (C.c_longlong * n)(*page),
                 (C.c_longlong * n)(*size), n, (C.c_int * m)(*[p[0] for p in pairs]), (C.c_int * m)(*[p[1] for p in pairs]), m, _lib.stream_ptr()),
               "copy_pages")
