"""How paged attention's work is cut and joined: equal shares, shares of a tile's own, many small tiles, long
tiles over many CTAs, lengths that change under a captured call, calls side by side."""
import numpy as np
import pytest
import torch

import marlin_q4 as mq
from test_gpu_attention import DEV, check, ints, make_cache, no_device_error, rand  # noqa: F401

pytestmark = pytest.mark.gpu


def wide(table, width):
    """The same pages in a table of more columns, its rows further apart than they are long."""
    t = torch.full((table.shape[0], width + 3), -1, dtype=torch.int32, device=DEV)
    t[:, :table.shape[1]] = table
    return t[:, :width]


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)]).tolist()


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4)])
def test_equal_shares_over_ragged_sequences(dim, bits):
    """More tiles than CTAs: a CTA works on several, a tile on up to two."""
    lens = ([0, 1, 16, 700, 33, 250, 17, 96] * 6)[:48]
    cache, table, ks, vs = make_cache(lens, 8, dim, bits, 16, 3)
    q = rand((48, 32, dim), 4, size=1.5)
    check(mq.paged_attention(q, cache, table, ints(lens)), q, ks, vs, lens, list(range(49)), dim ** -0.5)


@pytest.mark.parametrize("dim,bits,n_pos", [(64, 4, 70001), (128, 8, 9000), (256, 4, 5000)])
@pytest.mark.parametrize("width", [0, 40000])
def test_one_long_tile_over_many_ctas(dim, bits, n_pos, width):
    """Up to 274 partial rows of a tile; with a table far wider than the sequence the shares are equal ones."""
    cache, table, ks, vs = make_cache([n_pos], 1, dim, bits, 64, 5)
    if width:
        table = wide(table, width)
    q = rand((1, 3, dim), 6, size=1.5)
    check(mq.paged_attention(q, cache, table, ints([n_pos])), q, ks, vs, [n_pos], [0, 1], dim ** -0.5)


def test_small_work_under_a_wide_table():
    lens = [5, 0, 300, 64, 1]
    new = [2, 3, 4, 1, 4]
    cache, table, ks, vs = make_cache(lens, 2, 128, 4, 16, 8)
    q = rand((sum(new), 8, 128), 9, size=1.5)
    out = mq.paged_attention(q, cache, wide(table, 30000), ints(lens), ints(starts_of(new)), 4)
    check(out, q, ks, vs, lens, starts_of(new), 128 ** -0.5)
    assert not out[2:5].any()  # no position to see


def test_more_small_tiles_than_one_planning_pass():
    """1200 tiles of at most 40 rows: several per CTA, some without a position, some without a row."""
    new = [(3 * i) % 6 for i in range(300)]
    lens = [(7 * i) % 90 for i in range(300)]
    cache, table, ks, vs = make_cache(lens, 4, 64, 4, 32, 10)
    q = rand((sum(new), 32, 64), 11, size=1.5)
    out = mq.paged_attention(q, cache, table, ints(lens), ints(starts_of(new)), max(new))
    check(out, q, ks, vs, lens, starts_of(new), 0.125)


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 4), (256, 8)])
def test_long_tiles_over_many_ctas(dim, bits):
    """Two tiles of rows behind 20000 positions, each cut into some 74 parts."""
    new, n_pos = 20, 20011
    cache, table, ks, vs = make_cache([n_pos], 1, dim, bits, 64, 12)
    q = rand((new, 8, dim), 13, size=1.5)
    out = mq.paged_attention(q, cache, table, ints([n_pos]), ints([0, new]), new)
    check(out, q, ks, vs, [n_pos], [0, new], dim ** -0.5)


@pytest.mark.parametrize("dim,bits", [(64, 4), (256, 4)])
@pytest.mark.parametrize("most", [4, 64])
def test_captured_call_follows_lengths_and_starts(dim, bits, most):
    """Steps (4 x 4 rows) and chunks (64 x 4): replays equal plain calls, bit by bit."""
    top = [900, 333, 640, 257]
    cache, table, _, _ = make_cache(top, 2, dim, bits, 32, 14)
    q = rand((4 * most, 8, dim), 15, size=1.5)
    lens, starts = ints(top), ints([most * i for i in range(5)])
    out = torch.zeros_like(q)
    work = torch.empty(mq.attention_workspace_size(4 * most, 8, 2, dim, 4), dtype=torch.uint8, device=DEV)

    def run(out, work=None):
        return mq.paged_attention(q, cache, table, lens, starts, most, out=out, workspace=work)

    run(out, work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out, work)
    for n, s in ((top, [0, 1, 1, 3, 4]), ([0, 40, 64, 257], [0, most, most + 1, 2 * most, 2 * most]),
                 ([1, 333, 0, 9], [0, 1, 2, 3, 3 + most]), (top, [most * i for i in range(5)])):
        lens.copy_(ints(n))
        starts.copy_(ints(s))
        out.fill_(3.0)
        work.fill_(0xFF)
        graph.replay()
        want = run(torch.full_like(q, 3.0))
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
        assert (out[s[-1]:] == 3.0).all()
    del graph


def test_calls_side_by_side():
    """Steps and chunks on two streams, each with a workspace of its own."""
    lens = [1500, 77, 900]
    cache, table, _, _ = make_cache(lens, 2, 128, 4, 32, 16)
    new = {"steps": [2, 2, 2], "chunks": [130, 70, 200]}
    q = {k: rand((sum(n), 8, 128), 17 + len(k), size=1.5) for k, n in new.items()}
    cu = {k: ints(starts_of(n)) for k, n in new.items()}
    n = ints(lens)

    def run(k):
        return mq.paged_attention(q[k], cache, table, n, cu[k], max(new[k]))

    alone = {k: run(k) for k in new}
    torch.cuda.synchronize()
    streams = {k: torch.cuda.Stream() for k in new}
    got = {k: [] for k in new}
    for _ in range(10):
        for k, s in streams.items():
            with torch.cuda.stream(s):
                got[k].append(run(k))
    torch.cuda.synchronize()
    for k in new:
        for x in got[k]:
            assert torch.equal(x.view(torch.int16), alone[k].view(torch.int16))
