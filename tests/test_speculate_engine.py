"""KvCacheEngine's speculative step without a GPU: the structures of its calls, and what it refuses before them."""
import ctypes as C

import pytest

import runntime_b200._lib as L
from runntime_b200 import engine


@pytest.fixture
def step(monkeypatch):
    """An engine of three sequences on the CPU, and what its calls would be given."""
    torch = pytest.importorskip("torch")
    seen = []

    def rotary(ex, x, positions, plan, windows, **more):
        assert positions.dtype == torch.int32 and positions.numel() >= more["rows"]
        # what the kernel reads: rows numbers from the first address on
        seen.append(positions.as_strided((more["rows"],), (1,), positions.storage_offset()).tolist())

    monkeypatch.setattr(engine, "_bind_to_torch_stream", lambda ex: None)
    monkeypatch.setattr(engine, "rotary_batched", rotary)
    monkeypatch.setattr(engine, "tree_batched", lambda *a, **k: None)
    eng = engine.KvCacheEngine(None, batch=3, maxPositions=64, qHeads=2, kvHeads=1, headDim=8, device="cpu")
    eng.lens.copy_(torch.tensor([10, 20, 30]))
    eng.maxLen = 30
    eng.qkv = torch.zeros(12, 32, dtype=torch.float16)

    def call(depths, qkv=None):
        eng.stepTreeQkv(eng.qkv if qkv is None else qkv, None, None, depths, nodes=4)
        return seen[-1]

    call.engine, call.seen = eng, seen
    return call


def test_positions_are_rows_one_after_the_other(step):
    """Depths in any order in memory: the positions lie sequence by sequence."""
    torch = pytest.importorskip("torch")
    step.engine.setRotary(engine.RotaryPlan(8, None, 1.0))
    depths = torch.tensor([[0, 1, 1, 2], [0, 1, 2, 3], [0, 0, 1, 1]], dtype=torch.int32)
    want = [a + d for a, ds in zip((10, 20, 30), depths.tolist()) for d in ds]
    assert step(depths) == want
    assert step(depths.t().contiguous().t()) == want          # kept as [nodes, batch]
    assert step(depths.repeat_interleave(2, 1)[:, ::2]) == want
    for one in (depths[0], depths[:1], depths[0].expand(3, 4)):
        assert step(one) == [a + d for a in (10, 20, 30) for d in depths[0].tolist()]


def test_depths_of_another_shape_are_refused(step):
    torch = pytest.importorskip("torch")
    step.engine.setRotary(engine.RotaryPlan(8, None, 1.0))
    for shape in ((1,), (3,), (5,), (3, 1), (3, 3), (1, 3), (2, 4), (4, 3), (3, 5), (), (1, 3, 4)):
        with pytest.raises(ValueError, match="depths of shape"):
            step(torch.zeros(shape, dtype=torch.int32))
    with pytest.raises(ValueError, match="depths are torch.int64"):
        step(torch.zeros(4, dtype=torch.int64))
    assert not step.seen


def test_a_step_without_frequencies_is_refused(step):
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="setRotary"):
        step(torch.zeros(4, dtype=torch.int32))


def test_counted_commit_is_a_commit_and_an_address():
    assert L.CommitCountedArgs.layout == L.CommitArgs.layout + "P"
    assert L.CommitCountedArgs.committed.offset == C.sizeof(L.CommitArgs)
    for name, _ in L.CommitArgs._fields_:
        assert getattr(L.CommitCountedArgs, name).offset == getattr(L.CommitArgs, name).offset


@pytest.fixture
def commit(monkeypatch):
    """commitTree of an engine of three sequences on the CPU, with what its call would be given."""
    torch = pytest.importorskip("torch")
    seen = []
    monkeypatch.setattr(engine, "_bind_to_torch_stream", lambda ex: None)
    monkeypatch.setattr(engine, "commit_batched", lambda ex, caches, fresh, index, counts, lens, **more: seen.append(more))
    eng = engine.KvCacheEngine(None, batch=3, maxPositions=64, qHeads=2, kvHeads=1, headDim=8, device="cpu")

    def call(index, accepted, nodes=5, **more):
        eng.commitTree(0, 0, index, accepted, nodes=nodes, **more)
        return seen.pop()

    call.seen = seen
    call.ints = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype)
    return call


def test_indices_and_counts_that_a_commit_takes(commit):
    z = commit.ints
    assert commit(z(3, 4), z(3))["indexStride"] == 4
    assert commit(z(12), z(3))["indexStride"] == 4
    assert commit(z(3, 5), z(3), lead=0)["indexStride"] == 5
    assert commit(z(3, 9), z(3), indexStride=9)["indexStride"] == 9
    assert commit(z(3, 9)[:, :4], z(3), indexStride=9)["indexStride"] == 9
    assert commit(z(3, 9)[:, 2:6], z(4)[1:], indexStride=9)["indexStride"] == 9
    assert commit(z(3, 1), z(3), nodes=1)["indexStride"] == 1      # the leading rows alone
    assert commit(z(4, 4)[1:], z(3))["indexStride"] == 4
    assert commit(12345, 678)["indexStride"] == 4                  # addresses


def test_indices_and_counts_that_a_commit_refuses(commit):
    """64-bit numbers would be read as twice as many of 32 bits, rows further apart as rows of other sequences."""
    torch = pytest.importorskip("torch")
    z = commit.ints
    for bad, match in (((z(3, 4), z(3, dtype=torch.int64)), "accepted is torch.int64"),
                       ((z(3, 4, dtype=torch.int64), z(3)), "index is torch.int64"),
                       ((z(3, 4), z(3, dtype=torch.float32)), "accepted is torch.float32"),
                       ((z(3, 4), z(2)), "accepted of shape"), ((z(3, 4), z(6)[::2]), "accepted of shape"),
                       ((z(3, 3), z(3)), "index of shape"), ((z(2, 4), z(3)), "index of shape"),
                       ((z(3, 7), z(3)), "index of shape"), ((z(3, 8)[:, ::2], z(3)), "index of shape"),
                       ((z(4, 3).t(), z(3)), "index of shape"), ((z(11), z(3)), "index of shape")):
        with pytest.raises(ValueError, match=match):
            commit(*bad)
    with pytest.raises(ValueError, match="index of shape"):
        commit(z(3, 4), z(3), lead=0)
    with pytest.raises(ValueError, match="index of shape"):
        commit(z(3, 9), z(3), indexStride=8)
    assert not commit.seen


def test_masks_counts_and_sinks_that_a_step_takes_and_refuses(monkeypatch):
    torch = pytest.importorskip("torch")
    seen = []
    monkeypatch.setattr(engine, "_bind_to_torch_stream", lambda ex: None)
    monkeypatch.setattr(engine, "tree_batched", lambda *a, **k: seen.append(k))
    eng = engine.KvCacheEngine(None, batch=3, maxPositions=64, qHeads=4, kvHeads=2, headDim=8, device="cpu")

    def call(masks, **more):
        eng.stepTree(0, 0, 0, 0, masks, nodes=5, **more)
        seen.pop()

    def z(*shape, dtype=torch.int64):
        return torch.zeros(shape, dtype=dtype)

    i32, f32 = torch.int32, torch.float32
    call(z(3, 5))
    call(z(15))
    call(z(3, 5).view(torch.uint64))
    call(z(5), sharedMasks=True)
    call(z(3, 5), sharedMasks=True)
    call(z(5, 5)[1:4], nodeCounts=z(3, dtype=i32), sinks=z(4, dtype=f32))
    call(123, nodeCounts=456, sinks=789)
    for masks, more, match in ((z(3, 5, dtype=i32), {}, "masks is torch.int32"), (z(5), {}, "masks of shape"),
                               (z(3, 7), {}, "masks of shape"), (z(5, 3).t(), {}, "masks of shape"), (z(2, 5), {}, "masks of shape"),
                               (z(4), dict(sharedMasks=True), "masks of shape"),
                               (z(5).to("meta"), dict(sharedMasks=True), "masks is on meta"),
                               (z(3, 5), dict(nodeCounts=z(3)), "nodeCounts is torch.int64"),
                               (z(3, 5), dict(nodeCounts=z(2, dtype=i32)), "nodeCounts of shape"),
                               (z(3, 5), dict(sinks=z(4, dtype=torch.float16)), "sinks is torch.float16"),
                               (z(3, 5), dict(sinks=z(2, dtype=f32)), "sinks of shape")):
        with pytest.raises(ValueError, match=match):
            call(masks, **more)
    assert not seen


def test_a_plan_in_host_memory_is_refused():
    """rotary_plan's default device is torch's; a kernel cannot read from the CPU's."""
    pytest.importorskip("torch")
    for plan in (engine.rotary_plan(8), engine.rotary_plan(8, device="cpu")):
        with pytest.raises(ValueError, match="the plan is on cpu"):
            engine.rotary_batched(None, 16, 16, plan, [(0, 1, 16)], dtype="f16", rows=1, headDim=8, xRowStride=8)


def test_projections_of_another_type_or_layout_are_refused(step, monkeypatch):
    """Their rows are turned where they lie: in rows further apart, or of another type, that would be other memory."""
    torch = pytest.importorskip("torch")
    eng = step.engine
    eng.setRotary(engine.RotaryPlan(8, None, 1.0))
    depths = torch.zeros(4, dtype=torch.int32)
    committed = []
    monkeypatch.setattr(engine, "commit_batched", lambda *a, **k: committed.append(k))

    def commit(qkv):
        eng.commitTreeQkv(qkv, 0, 0, nodes=4)

    good = torch.zeros(12, 32, dtype=torch.float16)
    for qkv in (good, good.view(3, 4, 32), torch.zeros(13, 32, dtype=torch.float16)[1:]):
        step(depths, qkv)
        commit(qkv)
    assert len(step.seen) == len(committed) == 3
    for bad, match in ((good.float(), "qkv is torch.float32"), (torch.zeros(12, 64, dtype=torch.float16)[:, :32], "qkv of shape"),
                       (torch.zeros(32, 12, dtype=torch.float16).t(), "qkv of shape"), (good[:11], "qkv of shape"),
                       (torch.zeros(12, 40, dtype=torch.float16), "qkv of shape"), (good.to("meta"), "qkv is on meta")):
        with pytest.raises(ValueError, match="stepTreeQkv: " + match):
            step(depths, bad)
        with pytest.raises(ValueError, match="commitTreeQkv: " + match):
            commit(bad)
    assert len(step.seen) == len(committed) == 3
