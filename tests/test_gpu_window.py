"""Attention through a sliding window with sinks (wl_paged_window_attention) against 64 bits, over every cache."""
import numpy as np
import pytest

from windlass_amd import hip, paged

from . import paged_ref as P
from . import serving_ref as S
from .test_gpu_paged import random_trees

pytestmark = pytest.mark.gpu
TYPES = [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"), ("bf16", "mxfp4"), ("f32", "mxfp4")]
WINDOWS = [(1, 0), (1, 1), (2, 4), (31, 0), (32, 32), (33, 33), (64, 5), (100, 64), (500, 1), (700, 300), (5, 2 ** 32 - 1), (2 ** 32 - 1, 3)]


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_windows(gpu, window, sinks, q, cache):
    rng = np.random.default_rng(window % 1000 + sinks % 1000)
    lens, adds = [0, 1, 63, 130, 0, 517, 64, 2000], [1, 3, 0, 13, 5, 2, 64, 7]
    t = S.Serving(3, q, cache, 128, 32, 6, 16, lens, adds, random_trees(rng, adds), window=window, sinks=sinks, tail=2).upload().run()
    t.check()
    assert t.status() == 0


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("L,RP,H,ps", [(512, 64, 64, 64), (256, 32, 20, 8), (96, 8, 1, 1024), (512, 64, 16, 16)])
def test_shapes(gpu, L, RP, H, ps, q, cache):
    """Chains and single tokens, a window that leaves tiles out."""
    lens, adds = [900, 3, 300, 1500, 64], [40, 1, 9, 1, 64]
    S.Serving(L, q, cache, L, RP, H, ps, lens, adds, window=150, sinks=4, pad=8, row_pad=16).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("n", [0, 30, 31, 32, 33, 62, 63, 64, 65, 95, 96, 128, 300])
def test_one_token_around_tiles(gpu, q, cache, n):
    for window, sinks in ((32, 0), (33, 1), (31, 32), (64, 31)):
        S.Serving(n, q, cache, 128, 16, 16, 16, [n], [1], window=window, sinks=sinks).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_long_contexts(gpu, q, cache):
    """Walks of many tiles split over work-groups, windows of very uneven requests."""
    rng = np.random.default_rng(8)
    lens, adds = [20011, 5, 4700, 0, 9000], [1, 2, 64, 1, 3]
    S.Serving(9, q, cache, 128, 64, 8, 64, lens, adds, random_trees(rng, adds), window=4096, sinks=100).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_masks_that_are_no_trees(gpu, q, cache):
    """Any 64-bit mask: a node's position is the number of nodes it sees before its own. Some see nothing of the step."""
    rng = np.random.default_rng(12)
    lens, adds = [0, 70, 33, 3], [4, 4, 64, 64]
    masks = [0, 2, 0, 15] + [0, 8, 1, 0] + [int(x) for x in rng.integers(0, 1 << 62, 64)] + [0, (1 << 64) - 1] + \
        [1 << int(x) for x in rng.integers(0, 64, 62)]
    for window, sinks in ((3, 0), (20, 40), (80, 72)):
        S.Serving(13, q, cache, 256, 64, 6, 16, lens, adds, masks, window=window, sinks=sinks).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_a_window_over_everything_changes_nothing(gpu, q, cache):
    """Bit for bit the call without one where a context stands before the nodes; window 0 is none, whatever the sinks. (Of
    the request without a context, nodes that see nothing of the first 32 keys have their weights relative to the maximum
    of a later tile through a window, and to one above the walk's without: powers of two apart up to the maxima's own
    rounding, so their bits may differ, within the bound.)"""
    rng = np.random.default_rng(14)
    lens, adds = [700, 33, 0], [20, 1, 64]
    t = S.Serving(15, q, cache, 512, 64, 5, 32, lens, adds, random_trees(rng, adds)).upload().run()
    plain = t.out()
    for window, sinks in ((720, 0), (2 ** 32 - 1, 5), (0, 7), (1, 2 ** 31)):
        paged.window_attention(paged.WindowAttention(tree=t.args, window=window, n_sinks=sinks))
        hip.synchronize()
        assert np.array_equal(t.out()[:21], plain[:21])
        t.check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_pages_out_of_reach_are_not_looked_at(gpu, q, cache):
    """Their table entries name nothing of the cache; rows that the window passes over inside of tiles are NaN."""
    lens, adds, window, sinks, ps = [1000, 64, 517], [5, 1, 2], 70, 9, 16
    t = S.Serving(16, q, cache, 128, 32, 6, ps, lens, adds, window=window, sinks=sinks)
    table = t.table.copy()
    for r, (n, a) in enumerate(zip(lens, adds)):
        first = max(0, n - window + 1)  # the first node's first key
        for k in range(n):
            if sinks <= k < first:
                t.spoil(r, k)
        for page in range(-(-(n + a) // ps)):
            tiles = {k // 32 for k in range(page * ps, page * ps + ps)}
            if not tiles & ({k // 32 for k in range(sinks)} | {k // 32 for k in range(first, n + a)}):
                table[r, page] = [-1, t.n_pages, 2 ** 31 - 1, -2 ** 31][page % 4]
    assert (table != t.table).sum() > 30
    t.upload(table=table).run().check()
    assert t.status() == 0


@pytest.mark.parametrize("q,cache", TYPES)
def test_rows_that_some_nodes_may_not_see(gpu, q, cache):
    """A chain's deeper nodes have lost keys that its first ones see: a NaN there reaches the first ones alone."""
    n, a, window = 300, 40, 64
    for k in (n - window + 3, n - window + 30, 0):
        t = S.Serving(17, q, cache, 128, 32, 3, 16, [n], [a], window=window, sinks=1)
        t.spoil(0, k)
        t.upload().run()
        out = t.out()[:, :3 * 128].reshape(a, 3, 128)
        for i in range(a):
            if t.seen(0, i)[k]:
                assert np.isnan(out[i]).all()
            else:
                y, far = t.want(0, i)
                assert np.all(np.abs(out[i] - y) <= far)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("window,sinks", [(6000, 0), (2500, 1000)])
def test_walks_done_again(gpu, q, cache, window, sinks):
    """Scores that rise by more than a walk's first reference can hold."""
    lens, adds = [9000], [2]
    t = S.Serving(36, q, cache, 128, 16, 64, 16, lens, adds, spread=0.5, window=window, sinks=sinks)
    n = lens[0] + adds[0]
    t.qr[:, 0::16] = 128.0
    ramp = P.as_type((70.0 * (np.arange(n) % (11 * 32)) / 32 - 385) * np.log(2) / (128 * t.scale), "bf16")
    t.rows[0][:, 128] = ramp
    if t.mx:
        t.set_rows(t.rows)
    else:
        for k in range(n):
            t.pages[t.table[0, k // 16], k % 16, 128] = ramp[k]
    t.upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_refused_requests(gpu, q, cache):
    lens, adds = [200, 300, 9, 400], [2, 3, 1, 2]

    def tree():
        return S.Serving(17, q, cache, 128, 16, 6, 16, lens, adds, tail=3, window=50, sinks=2)
    t = tree()
    table = t.table.copy()
    table[1, 17] = t.n_pages  # inside of the window
    t.upload(table=table).run().check(nan=(1,))
    assert t.status() == paged.E_PAGE
    t = tree()
    t.upload(lens=[200, -5, 9, 2 ** 31 - 1]).run().check(nan=(1, 3))
    assert t.status() == paged.E_LEN
    t = tree()
    t.upload(cu=[0, 2, 5, 6, 12]).run().check(skip=(3,))
    assert t.status() == paged.E_LEN


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("R", [300, 1500, 4096])
def test_many_requests(gpu, R, q, cache):
    """More requests than a work-group has threads; some without tokens, some shorter than the window."""
    rng = np.random.default_rng(R)
    lens, adds = [int(x) for x in rng.integers(0, 300, R)], [int(x) for x in rng.integers(0, 3, R)]
    S.Serving(24, q, cache, 64, 8, 2, 8, lens, adds, random_trees(rng, adds), window=70, sinks=3).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("H,lens,adds", [(64, [2100, 40, 900, 1500, 2100, 3], [64, 60, 64, 64, 64, 64]), (64, list(range(40, 1240, 20)), [5, 9, 1, 8] * 15),
                                         (16, list(range(0, 3000, 100)) + [50] * 40, [1] * 30 + [0] * 40)], ids=["chunks", "rows", "singles"])
def test_splits(gpu, H, lens, adds, window, q, cache):
    """More row tiles than work-groups, in chunks and whole; single row tiles in pieces, among requests without tokens."""
    rng = np.random.default_rng(31)
    S.Serving(32, q, cache, 32, 8, H, 16, lens, adds, random_trees(rng, adds), window=window, sinks=5).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("window,sinks", [(128, 0), (90, 0), (200, 40)])
def test_chains_whose_last_node_begins_with_a_tile(gpu, window, sinks, q, cache):
    """It sees nothing of the tile before it, with which the request's walk begins; lengths around those, too."""
    lens, adds = [], []
    for a in (2, 8, 33):
        for off in (-16, -1, 0, 1, 16):
            lens.append(32 * 11 + window - a + off)
            adds.append(a)
    S.Serving(33, q, cache, 128, 32, 6, 16, lens, adds, window=window, sinks=sinks).upload().run().check()
