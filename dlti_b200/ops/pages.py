"""Copies of cache pages (csrc/pages.cu): what a sequence that goes on from another one's tokens needs of its own."""
from __future__ import annotations

import ctypes as C
from array import array

import torch

from . import _lib

_call = None


def _bind():
    global _call
    _call = _lib.fn("dlti_copy_pages", [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p])
    return _call


def check_copies(src: list[int], dst: list[int], num_pages: int) -> tuple[list[int], list[int]]:
    """The sources and destinations of a call, without those that copy a page onto itself. Refused: pages outside the cache, a page written twice, a
    page both read and written (copies have no order)."""
    if len(src) != len(dst):
        raise ValueError(f"copy_pages: {len(src)} sources for {len(dst)} destinations")
    if not src:
        return src, dst
    if min(src) < 0 or min(dst) < 0 or max(src) >= num_pages or max(dst) >= num_pages:
        raise ValueError(f"copy_pages: pages are 0 .. {num_pages - 1}")
    written = set(dst)
    if len(written) < len(dst):
        raise ValueError("copy_pages: a page is written twice")
    if not written.isdisjoint(src):
        pairs = [(a, b) for a, b in zip(src, dst) if a != b]
        src, dst = [a for a, _ in pairs], [b for _, b in pairs]
        if not set(dst).isdisjoint(src):
            raise ValueError("copy_pages: a page is both read and written")
    return src, dst


def _page(t: torch.Tensor, page_dim: int) -> tuple[int, ...]:
    """(layers, bytes from layer to layer, bytes from page to page, bytes of a page) of a cache; () if nothing is in it."""
    shape, stride, es = t.shape, t.stride(), t.element_size()
    if t.is_contiguous():                                    # as all that hold nothing are
        if not t.numel():
            return ()
        return (shape[0], stride[0] * es, stride[1] * es, stride[1] * es) if page_dim else (1, 0, stride[0] * es, stride[0] * es)
    n = 1
    for d in range(len(shape) - 1, page_dim, -1):
        if shape[d] != 1 and stride[d] != n:
            raise ValueError("copy_pages: what a page holds is contiguous")
        n *= shape[d]
    if shape[page_dim] > 1 and stride[page_dim] < n:
        raise ValueError("copy_pages: pages do not overlap")
    return (shape[0], stride[0] * es, stride[1] * es, n * es) if page_dim else (1, 0, stride[0] * es, n * es)


def copy_pages(caches: list[torch.Tensor], src: list[int], dst: list[int], page_dim: int = 0) -> None:
    """Pages src[i] -> dst[i] (whole numbers on the host) of every tensor in `caches`: [pages, ...], or with page_dim=1 [layers, pages, ...]. What a
    page holds is contiguous. One launch for up to 32 tensors and 300 pairs; the pairs travel with it, so a graph that captures the call replays
    these."""
    if page_dim not in (0, 1):
        raise ValueError("copy_pages: pages are dimension 0, or dimension 1 behind the layers")
    if not caches:
        return
    num = caches[0].shape[page_dim]
    for t in caches:
        if t.shape[page_dim] != num:
            raise ValueError(f"copy_pages: caches of {num} and {t.shape[page_dim]} pages")
    src, dst = check_copies(src, dst, num)
    flat = []
    for t in caches:
        page = _page(t, page_dim)
        if page:
            flat.append(t.data_ptr())
            flat += page
    if not src or not flat:
        return
    if not caches[0].is_cuda:
        a, b = torch.tensor(src), torch.tensor(dst)
        for t in caches:
            if page_dim == 0:
                t[b] = t[a]
            else:
                t[:, b] = t[:, a]
        return
    d = torch.cuda.current_device()
    for t in caches:
        if t.get_device() != d:
            raise ValueError(f"copy_pages: every cache is on the current device, cuda:{d}")
    f = _call or _bind()
    what, a, b = array("q", flat), array("i", src), array("i", dst)
    _lib.check(f(what.buffer_info()[0], len(flat) // 5, a.buffer_info()[0], b.buffer_info()[0], len(a), torch._C._cuda_getCurrentRawStream(d)),
               "copy_pages")
