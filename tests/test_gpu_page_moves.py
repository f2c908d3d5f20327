"""Page copies inside a pool (bikv_copy_pages): byte-exact against a numpy restatement, for every kind of pool."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bk(lib):
    import bikv_pagecopy
    return bikv_pagecopy


def _moves(rng, n_pages, n):
    ids = rng.permutation(n_pages)
    return ids[:n].copy(), ids[n:2 * n].copy()


def _bytes(rng, shape):
    return rng.integers(0, 256, size=shape, dtype=np.uint8)


@pytest.mark.parametrize("tile", [1, 3, 32, 100, 512, 1024, 1040, 4096, 16384, 40000])
@pytest.mark.parametrize("scale_tile", [0, 4, 12, 32])
def test_every_tile_size(bk, cuda, tile, scale_tile):
    rng = np.random.default_rng(tile * 37 + scale_tile)
    planes, pages, n = 3, 41, 17
    host = _bytes(rng, (planes, pages, tile))
    dev = torch.from_numpy(host).to(cuda)
    shost = _bytes(rng, (planes, pages, scale_tile)) if scale_tile else None
    sdev = torch.from_numpy(shost).to(cuda) if scale_tile else None
    pool = bk.PagedKVPool.from_stacked(dev, plane_dims=1, scale=sdev)
    src, dst = _moves(rng, pages, n)
    src[3] = src[0]                                   # a source may repeat: two forks of one page
    pool.copy_pages(*pool.page_moves(src, dst))
    pool.check()
    host[:, dst] = host[:, src]
    assert np.array_equal(dev.cpu().numpy(), host)
    if scale_tile:
        shost[:, dst] = shost[:, src]
        assert np.array_equal(sdev.cpu().numpy(), shost)


def test_pools_with_k_and_v_adjacent_and_token_by_token(bk, cuda):
    rng = np.random.default_rng(5)
    src, dst = _moves(rng, 30, 12)
    a = [torch.randn(30, 2, 16, 2, 64, device=cuda).half() for _ in range(3)]
    want = [t.clone() for t in a]
    pool = bk.PagedKVPool.from_layers_kv_adjacent(a)
    pool.copy_pages(*pool.page_moves(src, dst))
    pool.check()
    for t, w in zip(a, want):
        w[dst] = w[src]
        assert torch.equal(t, w)
    for block in (16, 5):
        b = [torch.randn(30 * block, 2, 2, 128, device=cuda).half() for _ in range(2)]
        want = [t.clone().view(30, block, 2, 2, 128) for t in b]
        pool = bk.PagedKVPool.from_token_kv_layers(b, block)
        pool.copy_pages(*pool.page_moves(src, dst))
        pool.check()
        for t, w in zip(b, want):
            w[dst] = w[src]
            assert torch.equal(t.view(w.shape), w)


def test_a_bad_id_is_reported_and_the_others_are_copied(bk, cuda):
    host = np.arange(2 * 10 * 64, dtype=np.uint8).reshape(2, 10, 64)
    dev = torch.from_numpy(host.copy()).to(cuda)
    pool = bk.PagedKVPool.from_stacked(dev, plane_dims=1)
    src = torch.tensor([0, 99, 2, -1, 4], device=cuda)
    dst = torch.tensor([5, 6, 10, 7, 8], device=cuda)
    pool.copy_pages(src, dst)
    with pytest.raises(RuntimeError, match="page-id"):
        pool.check()
    host[:, 5], host[:, 8] = host[:, 0], host[:, 4]
    assert np.array_equal(dev.cpu().numpy(), host)
    pool.check()


def test_a_page_onto_itself_and_nothing_at_all(bk, cuda):
    dev = torch.randn(2, 6, 128, device=cuda)
    was = dev.clone()
    pool = bk.PagedKVPool.from_stacked(dev, plane_dims=1)
    pool.copy_pages(*pool.page_moves([3, 1], [3, 2]))
    pool.copy_pages(*pool.page_moves([], []))
    pool.check()
    was[:, 2] = was[:, 1]
    assert torch.equal(dev, was)


def test_refusals(bk, lib, cuda):
    from bikv_pagecopy import _lib
    pool = bk.PagedKVPool.from_stacked(torch.zeros(2, 8, 64, device=cuda), plane_dims=1)
    for src, dst, what in (([0, 1], [2], "length"), ([0, 1], [2, 2], "more than once"), ([0, 1], [1, 2], "source and a destination"),
                           ([0], [8], "outside"), ([-1], [3], "outside")):
        with pytest.raises(RuntimeError, match=what):
            pool.page_moves(src, dst)
    ids = torch.arange(4, device=cuda)
    for bad in (ids.int(), ids.cpu(), ids.view(2, 2), torch.arange(8, device=cuda)[::2]):
        with pytest.raises(RuntimeError):
            pool.copy_pages(bad, ids)
        with pytest.raises(RuntimeError):
            pool.copy_pages(ids, bad)
    with pytest.raises(RuntimeError, match="length"):
        pool.copy_pages(ids, ids[:2])
    assert lib.bikv_copy_pages(None, None, None, 0, None) == _lib.EINVAL
    assert lib.bikv_copy_pages(pool._h, None, None, -1, None) == _lib.EINVAL
    assert lib.bikv_copy_pages(pool._h, None, None, 3, None) == _lib.EINVAL
    assert lib.bikv_copy_pages(pool._h, None, None, 0, None) == _lib.OK
    bk.set_tuning(debug_unique=1)
    with pytest.raises(RuntimeError, match="more than once"):
        pool.copy_pages(ids[:2], torch.tensor([5, 5], device=cuda))


def test_replays_from_a_graph_on_another_stream(bk, cuda):
    dev = torch.randint(0, 255, (4, 50, 2048), dtype=torch.uint8, device=cuda)
    pool = bk.PagedKVPool.from_stacked(dev, plane_dims=1)
    rng = np.random.default_rng(0)
    src, dst = pool.page_moves(*_moves(rng, 50, 20))
    pool.copy_pages(src, dst)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        pool.copy_pages(src, dst)
    for i in range(3):
        s, d = pool.page_moves(*_moves(rng, 50, 20))
        src.copy_(s)
        dst.copy_(d)
        dev.random_(0, 255)
        want = dev.clone()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want[:, d] = want[:, s]
        assert torch.equal(dev, want), i
    pool.check()


def test_planes_beyond_4_gib(bk, cuda):
    """Byte offsets inside a plane pass 32 bits."""
    pages, tile = 70000, 65536
    dev = torch.empty((1, pages, tile), dtype=torch.uint8, device=cuda)
    scale = torch.empty((1, pages, 8), dtype=torch.float32, device=cuda)
    pool = bk.PagedKVPool.from_stacked(dev, plane_dims=1, scale=scale)
    src, dst = [3, 69999, 65535], [69998, 4, 65536]
    for p in src:
        dev[0, p].random_(0, 255)
        scale[0, p].normal_()
    pool.copy_pages(*pool.page_moves(src, dst))
    pool.check()
    for s, d in zip(src, dst):
        assert torch.equal(dev[0, s], dev[0, d]) and torch.equal(scale[0, s], scale[0, d])
