"""paged_attention on metadata that leaves the table: which keys there are, and what a row sees of them, as cutile_hip.h has it."""
import pytest
import torch

import paged_ref as ref
from paged_ref import Batch
from test_paged_attention import problem
from test_paged_tiles import TILES, name
from test_paged_weights import bound


def compare(ct, dev, b, held, heads, group, d, mx, window, wrong_pages=()):
    """launches for lengths `held` on b's table, in tiles of every number of rows, against 64 bits"""
    q, k, v, scales, real = problem(b, heads, group, d, "f16", mx, dev)
    b.held, b.lens = held, torch.tensor(held, dtype=torch.int32)
    for at, page in wrong_pages:
        b.table[at] = page
    parts = ref.attention(b, q, *real, float(torch.tensor(d ** -0.5, dtype=torch.float32)), window)
    tol = bound(q.dtype, parts, d, b.table.shape[1] * b.page)
    for rows in (None, *TILES[d]):
        for kw in ({}, {"max_new": max(b.new), "max_context": 64}):
            out = torch.full_like(q, 9.0).to(dev)
            ct.paged_attention(q.to(dev), k, v, *b.where(dev), ct.partition(out, [1, 1, d]), d ** -0.5, window=window, variant=rows and name("f16", mx, d, rows), **scales, **kw)
            assert bool(((out.cpu().double() - parts[0]).abs() <= tol).all()), (rows, kw)
    return parts[0]


@pytest.mark.gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d,group", [(64, 1), (128, 4), (256, 2)])
@pytest.mark.parametrize("window", [1, 40, 1000, 2 ** 31 - 1])
def test_gpu_windows_at_the_largest_lengths(ct, dev, mx, d, group, window):
    """rows at positions next to 2^31, whose window lies behind the table or reaches into it"""
    b = Batch([3, 1, 50, 40], [64] * 4, 16, table_pages=4, seed=d)
    want = compare(ct, dev, b, [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 1, 1040], 2, group, d, mx, window)
    assert bool((want[:54] == 0).all()) == (window < 2 ** 31 - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d,group", [(64, 1), (128, 4), (256, 2)])
@pytest.mark.parametrize("window", [0, 3, 40])
def test_gpu_lengths_that_leave_the_table(ct, dev, mx, d, group, window):
    """keys behind the table do not exist: rows behind it attend to those in front of its end that their window reaches; rows in front of position 0 are zeros; a page that
    the cache lacks holds zeros, which count"""
    b = Batch([2, 50, 4, 60, 1, 3], [64, 64, 64, 64, 40, 64], 16, table_pages=4, seed=window + d)
    want = compare(ct, dev, b, [66, 90, 2, 30, -7, 2 ** 31 - 1], 2, group, d, mx, window, [((0, 2), -1), ((1, 0), b.pages)])   # (the third and fourth have fewer tokens than new ones)
    assert bool((want[52:54] == 0).all()) and bool((want[54:56] != 0).all()) and bool((want[56:86] == 0).all()) and bool((want[116] == 0).all())
    assert bool((want[117:] == 0).all()) == (window > 0) and bool((want[0] != 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("d,group", [(64, 4), (128, 4), (256, 2)])
def test_gpu_several_streams_and_graphs_at_once(ct, dev, d, group):
    """launches that share keys on two streams (a workspace of each stream's own) beside two graphs (one of the caller's each): the bits of each by itself"""
    work = []
    for i, (new, held) in enumerate([([1, 1], [9000, 4000]), ([150, 3], [5000, 2000]), ([1, 1, 1], [3000, 8000, 10]), ([40], [6000])]):
        b = Batch(new, held, 16, seed=i)
        q, k, v, _, _ = problem(b, 2, group, d, "bf16", False, dev)
        work.append((b, q.to(dev), k, v, b.where(dev), torch.zeros_like(q, device=dev)))

    def launch(i, workspace=None, stream=None):
        b, q, k, v, where, out = work[i]
        ct.paged_attention(q, k, v, *where, ct.partition(out, [1, 1, d]), d ** -0.5, max_new=max(b.new), max_context=max(b.held), workspace=workspace, stream=stream)

    alone = []
    for i in range(4):
        launch(i)
        torch.cuda.synchronize()
        alone.append(work[i][-1].clone())
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [torch.zeros(ct.PAGED_ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device=dev) for _ in range(2)]
    torch.cuda.synchronize()
    graphs = [ct.CapturedGraph().capture(lambda s, i=i: launch(2 + i, spaces[i], s)) for i in range(2)]
    for _ in range(5):
        for w in work:
            w[-1].fill_(5.0)
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                graphs[i].launch()
                with torch.cuda.stream(streams[i]):
                    launch(i)
        for g in graphs:
            g.synchronize()
        torch.cuda.synchronize()
        for w, want in zip(work, alone):
            assert torch.equal(w[-1], want)
    for g in graphs:
        g.close()
