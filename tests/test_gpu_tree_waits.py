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
