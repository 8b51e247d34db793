"""Waits inside tree attention that run out: an error status, and nothing left behind for the calls after it."""
import pytest

from gpu_harness import ex  # noqa: F401
from test_gpu_speculate import Tree, on_torch  # noqa: F401

pytestmark = pytest.mark.gpu
DEFAULT = 1 << 20
# one stream to a warpgroup, heads at columns of their own, and four row tiles
CASES = [((8, 2, 128), 25), ((8, 8, 52), 7), ((8, 1, 128), 64)]


@pytest.fixture
def polls(on_torch):
    from runntime_b200._lib import OPT_WAIT_POLLS
    yield lambda n: on_torch.setOption(OPT_WAIT_POLLS, n)
    on_torch.setOption(OPT_WAIT_POLLS, DEFAULT)


def gives_up(ex):
    from runntime_b200 import RunntimeError
    with pytest.raises(RunntimeError, match="wait ran out"):
        ex.sync()


@pytest.mark.parametrize("shape,nodes", CASES)
def test_tree_gives_up(on_torch, polls, shape, nodes):
    """A limit of one poll, which does not wait for anything: the call ends, and says so.  What was on its way
    has arrived before its block has ended: the call after it, in the same shared and tensor memory, is right."""
    t = Tree("f16", *shape, nodes, [3000, 77, 1500], seed=nodes)
    want = t.call(on_torch, splits=1).clone()
    on_torch.sync()
    t.check(want)
    for _ in range(10):
        polls(1)
        t.call(on_torch, splits=1)
        polls(DEFAULT)
        t.out.fill_(7.0)
        got = t.call(on_torch, splits=1)
        gives_up(on_torch)             # (of the call before)
        assert t.torch.equal(got, want)
    on_torch.sync()


@pytest.mark.parametrize("shape,nodes", CASES)
def test_tree_gives_up_before_the_joining_launch(on_torch, polls, shape, nodes):
    """The launch that joins the parts comes after one that has given up, and finds another call's floats where the
    places of the parts would be: it joins nothing outside of its scratch."""
    other = Tree("f32", 8, 2, 64, 64, [2000] * 8, seed=9)
    t = Tree("f16", *shape, nodes, [20000, 9000, 15000], seed=nodes)    # (more tiles to a run than a ring has places)
    want = t.call(on_torch, splits=5).clone()
    on_torch.sync()
    t.check(want)
    for _ in range(5):
        other.call(on_torch, splits=64)     # partial results all over the scratch
        polls(1)
        t.call(on_torch, splits=5)
        polls(DEFAULT)
        t.out.fill_(7.0)
        got = t.call(on_torch, splits=5)
        gives_up(on_torch)
        assert t.torch.equal(got, want)
    on_torch.sync()


def test_tree_rows_computed_again_hold_up_no_wait(on_torch, polls):
    """One infinite value in a long cache, seen by 32 rows of every warp, with short sequences after it in the same streams:
    the rows take milliseconds to compute again, the limit here, and nobody has to wait for them."""
    lens = [4000] + [64] * 79
    t = Tree("f16", 32, 8, 16, 32, lens, seed=2)
    t.v[0, 5] = float("inf")
    polls(2000)
    got = t.call(on_torch, splits=1)
    on_torch.sync()                      # (no wait has run out)
    got = got.view(80, -1)
    assert (got[0] == float("inf")).all()
    t.check(got, sequences=range(1, 80))
    # cut anywhere
    t.out.fill_(7.0)
    got = t.call(on_torch, splits=5).view(80, -1)
    on_torch.sync()
    assert (got[0] == float("inf")).all()
    t.check(got, sequences=range(1, 80))


@pytest.mark.parametrize("shape", [(8, 2, 128), (8, 8, 52), (4, 2, 40), (6, 6, 36), (8, 1, 64)])
@pytest.mark.parametrize("splits", [1, 5])
def test_tree_rows_that_see_what_is_not_finite(on_torch, shape, splits):
    """What a row sees decides, column by column; heads beside it and other sequences stay as they are, to the bit."""
    inf, nan = float("inf"), float("nan")
    H, K, D = shape
    G, T = H // K, 17
    t = Tree("f16", *shape, T, [700, 130], seed=8)
    torch = t.torch
    clean = t.call(on_torch, splits=splits).clone()
    on_torch.sync()
    t.check(clean)

    def parts(x):       # [sequence, node, kv head, query head of it, column]
        return x.view(2, T, K, G, D)

    def after(spoil):
        kept = [x.clone() for x in (t.q, t.k, t.v, t.kNew, t.vNew)]
        spoil()
        t.out.fill_(7.0)
        got = t.call(on_torch, splits=splits).clone()
        on_torch.sync()
        for x, y in zip((t.q, t.k, t.v, t.kNew, t.vNew), kept):
            x.copy_(y)
        return parts(got)

    was = parts(clean)
    others = [h for h in range(K) if h != 0]

    def near(a, b):     # two roundings, and another order of the sums
        a, b = a.double(), b.double()
        return bool(((a - b).abs() <= 2.0 ** -10 * b.abs() + 2.0 ** -11).all())

    # infinite values of one column of head 0, in the cache
    def values():
        t.v[0, 5, 3] = inf
    got = after(values)
    assert torch.equal(got[1], was[1]) and torch.equal(got[0][:, others], was[0][:, others])
    assert (got[0][:, 0, :, 3] == inf).all()
    rest = [c for c in range(D) if c != 3]
    assert near(got[0][:, 0][..., rest], was[0][:, 0][..., rest])

    def both():
        t.v[0, 5, 3], t.v[0, 600, 3], t.v[0, 9, 1] = inf, -inf, -inf
    got = after(both)
    assert torch.equal(got[1], was[1]) and torch.equal(got[0][:, others], was[0][:, others])
    assert got[0][:, 0, :, 3].isnan().all() and (got[0][:, 0, :, 1] == -inf).all()
    assert near(got[0][:, 0, :, 0], was[0][:, 0, :, 0])

    # a key of head 0: its rows have no value, others do, although they lie in the same tiles where heads are narrow
    for value in (nan, inf):
        def key():
            t.k[0, 400, :D] = value
        got = after(key)
        assert torch.equal(got[1], was[1])
        assert got[0][:, 0].isnan().all()       # (products of infinities of both signs, too)
        if D % 8 == 0:
            assert torch.equal(got[0][:, others], was[0][:, others])
        else:           # (computed again, key by key)
            assert near(got[0][:, others], was[0][:, others])

    # a query of one node and head
    def query():
        t.q[3, :D] = nan
    got = after(query)
    assert got[0, 3, 0, 0].isnan().all()
    got[0, 3, 0, 0] = was[0, 3, 0, 0]
    assert torch.equal(got, was)
