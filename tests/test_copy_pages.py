"""Copies of cache pages: every layer, any page size and alignment; what a call refuses."""
import pytest
import torch

from dlti_b200.ops.pages import check_copies, copy_pages

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def filled(shape, seed, dev, dtype=torch.uint8):
    n = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
    return torch.randint(0, 256, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8).view(dtype).view(shape).to(dev)


def bytes_of(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("page", [(16, 2, 128), (1,), (5,), (3, 4), (2, 16, 700), (16, 32, 128)])
@pytest.mark.parametrize("pairs", [1, 7, 300, 301])
def test_pages_of_layers(dev, page, pairs):
    """One tensor with all layers and one tensor a layer; pages of one byte to several pieces; more pairs than one launch takes."""
    if pairs > 7 and torch.Size(page).numel() > 20000:
        pairs = 9
    n = 2 * pairs + 3
    order = torch.randperm(n, generator=torch.Generator().manual_seed(pairs)).tolist()
    src, dst = [order[i // 2] for i in range(pairs)], order[pairs:2 * pairs]      # a page may be read more than once
    a, b = filled((3, n, *page), 1, dev), filled((3, n, 2), 2, dev, torch.float32)
    wa, wb = a.clone(), b.clone()
    for x, y in zip(src, dst):
        wa[:, y], wb[:, y] = a[:, x], b[:, x]
    copy_pages([a, b], src, dst, page_dim=1)
    assert torch.equal(a, wa) and torch.equal(bytes_of(b), bytes_of(wb))
    each = [filled((n, *page), 3 + i, dev) for i in range(35 if pairs < 10 else 2)]   # more tensors than one launch takes
    want = [t.clone() for t in each]
    for x, y in zip(src, dst):
        for t, w in zip(each, want):
            w[y] = t[x]
    copy_pages(each, src, dst)
    assert all(torch.equal(t, w) for t, w in zip(each, want))


@pytest.mark.parametrize("dev", DEVICES)
def test_unaligned_and_strided(dev):
    """Caches that begin anywhere and whose pages are further apart than they are long; neighbours stay as they were."""
    room = filled((2, 9, 40), 1, dev)
    want = room.clone()
    a = room[:, :, 3:36]
    want[:, 5, 3:36], want[:, 0, 3:36] = room[:, 2, 3:36], room[:, 8, 3:36]
    copy_pages([a], [2, 8, 4], [5, 0, 4], page_dim=1)
    assert torch.equal(room, want)
    copy_pages([a], [], [], page_dim=1)
    copy_pages([], [1], [2])
    assert torch.equal(room, want)


def test_refusals():
    a = torch.zeros(3, 8, 4)
    for src, dst in (([0], [8]), ([-1], [2]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0, 1], [1, 0])):
        with pytest.raises(ValueError):
            copy_pages([a], src, dst, page_dim=1)
    for caches, dim in (([a, torch.zeros(3, 9, 4)], 1), ([a], 2), ([a.transpose(0, 2)], 1), ([a[:, :1].expand(3, 8, 4)], 1)):
        with pytest.raises(ValueError):
            copy_pages(caches, [0], [1], page_dim=dim)
    assert check_copies([1, 2, 2], [1, 3, 4], 5) == ([2, 2], [3, 4])


@pytest.mark.parametrize("dev", DEVICES)
def test_caches_of_nothing(dev):
    """Caches without layers, pages without numbers and caches without pages beside others: nothing of them is copied, the others are."""
    a = filled((3, 5, 40), 1, dev)
    want = a.clone()
    want[:, 4], want[:, 0] = a[:, 1], a[:, 2]
    empty = [torch.zeros(s, device=dev) for s in ((0, 5, 8), (3, 5, 0), (3, 5, 4, 0, 2))]
    copy_pages([empty[0], a, *empty[1:]], [1, 2], [4, 0], page_dim=1)
    assert torch.equal(a, want)
    copy_pages(empty, [1, 2], [4, 0], page_dim=1)
    copy_pages([torch.zeros((0, 4), device=dev)], [], [])
    with pytest.raises(ValueError):
        copy_pages([torch.zeros((3, 0, 4), device=dev)], [0], [1], page_dim=1)
