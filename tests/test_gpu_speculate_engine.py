"""KvCacheEngine's speculative step where sequences are refused."""
import pytest

from gpu_harness import ex  # noqa: F401
from test_gpu_speculate import gen, on_torch, torch_  # noqa: F401

pytestmark = pytest.mark.gpu


def dev(x):
    return torch_().tensor(x, dtype=torch_().int32, device="cuda")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("lead,index,accepted,refused", [
    (1, [[0, 1, 2], [0, 3, 1], [2, 0, 0]], [2, 2, 1], [1]),       # an index past the last node
    (1, [[0, 1, 2], [-1, 0, 1], [2, 0, 0]], [2, 3, 0], [1]),      # a path's filling counted as a node
    (1, [[0, 1, 2], [0, 1, 2], [0, 1, 2]], [3, 4, 1], [1]),       # more than there are nodes
    (1, [[0, 1, 2], [0, 1, 2], [0, 1, 2]], [0, -2, 3], [1]),      # negative
    (0, [[0, 1, 2, 3], [0, 4, 2, 3], [3, 2, 1, 0]], [0, 2, 4], [1]),
])
def test_lengths_grow_by_what_was_committed(on_torch, dtype, lead, index, accepted, refused):
    """A refused sequence keeps its rows and its length; the next step still has it as it was."""
    from runntime_b200 import RunntimeError, engine
    torch = torch_()
    B, T, w, most = 3, 4, 128, 16
    eng = engine.KvCacheEngine(on_torch, batch=B, maxPositions=most, qHeads=2, kvHeads=2, headDim=64, dtype=dtype)
    k, v = (torch.randn(B * T, w, generator=gen(i), device="cuda").to(eng.k.dtype) for i in (1, 2))
    eng.lens.copy_(dev([5, 7, 0]))
    eng.maxLen = 7
    eng.commitTree(k, v, dev(index), dev(accepted), nodes=T, lead=lead)
    with pytest.raises(RunntimeError, match="status"):
        on_torch.sync()
    want = [n + (0 if b in refused else lead + accepted[b]) for b, n in enumerate([5, 7, 0])]
    assert eng.lens.tolist() == want
    assert eng.committed.tolist() == [a - b for a, b in zip(want, [5, 7, 0])]
    for cache, fresh in ((eng.k, k), (eng.v, v)):
        for b, was in enumerate([5, 7, 0]):
            rows = [] if b in refused else [*range(lead), *(lead + i for i in index[b][:accepted[b]])]
            assert torch.equal(cache[b, was:was + len(rows)], fresh.view(B, T, w)[b, rows])
            assert (cache[b, was + len(rows):] == 0).all() and (cache[b, :was] == 0).all()


def test_a_full_cache_keeps_its_length(on_torch):
    """Rows that do not fit, as a replayed step meets them: nothing is written and no length passes the capacity."""
    from runntime_b200 import RunntimeError, engine
    torch = torch_()
    B, T, w, most = 3, 4, 128, 10
    eng = engine.KvCacheEngine(on_torch, batch=B, maxPositions=most, qHeads=2, kvHeads=2, headDim=64)
    x = torch.randn(B * T, w, generator=gen(3), device="cuda").half()
    eng.lens.copy_(dev([8, 3, 7]))
    before = [c.clone() for c in (eng.k, eng.v)]
    eng.commitTree(x, x, dev([[0, 1, 2]] * B), dev([2, 2, 2]), nodes=T)
    with pytest.raises(RunntimeError, match="status"):
        on_torch.sync()
    assert eng.lens.tolist() == [8, 6, 10]
    for c, was in zip((eng.k, eng.v), before):
        assert torch.equal(c[0], was[0])
        assert torch.equal(c[1, 3:6], x.view(B, T, w)[1, :3]) and torch.equal(c[2, 7:], x.view(B, T, w)[2, :3])
    eng.commitTree(x, x, dev([[0, 1, 2]] * B), dev([1, 0, -1]), nodes=T, lead=1)    # (one fits to the last row)
    with pytest.raises(RunntimeError, match="status"):
        on_torch.sync()
    assert eng.lens.tolist() == [10, 7, 10]


def test_committed_rows_of_many_tensors(on_torch):
    """More tensors than one launch takes: the count is the same from each."""
    from runntime_b200 import RunntimeError, engine
    torch = torch_()
    B, T, w = 2, 3, 8
    caches = torch.zeros(130, B, 9, w, device="cuda")
    fresh = torch.randn(130, B * T, w, generator=gen(4), device="cuda")
    committed = dev([77, 77])
    engine.commit_batched(on_torch, caches, fresh, dev([[0, 1], [0, 2]]), dev([2, 2]), dev([6, 1]), dtype="f32", batch=B, nodes=T,
                          cacheRows=9, width=w, lead=1, indexStride=2, committed=committed)
    with pytest.raises(RunntimeError, match="status"):
        on_torch.sync()
    assert committed.tolist() == [3, 0]
    assert torch.equal(caches[:, 0, 6:], fresh.view(130, B, T, w)[:, 0]) and (caches[:, 1] == 0).all()


def test_a_step_is_captured_when_the_bound_is_full(on_torch):
    """The host's bound of the lengths has met the capacity, the lengths have not: they cannot be asked for under a capture,
    and the step is captured all the same; replays go on until the rows no longer fit, and say so."""
    import runntime_b200 as rt
    from runntime_b200 import RunntimeError, engine
    torch = torch_()
    T, w, most = 8, 128, 24
    masks = torch.tensor(engine.tree_masks([-1] + [0] * 7), device="cuda")
    x = torch.randn(2 * T, w, generator=gen(1), device="cuda").half()
    index, accepted = torch.zeros(2, T - 1, dtype=torch.int32, device="cuda"), dev([1, 0])
    outs = []
    e = rt.CudaExecutor(0)
    try:
        engines = [engine.KvCacheEngine(ex, batch=2, maxPositions=most, qHeads=2, kvHeads=2, headDim=64) for ex in (on_torch, e)]
        for eng in engines:
            out = torch.empty_like(x)
            outs.append(out)
            for _ in range(3):
                eng.stepTree(x, x, x, out, masks, nodes=T, sharedMasks=True)
                eng.commitTree(x, x, index, accepted, nodes=T)
            assert eng.maxLen == most and eng.lens.tolist() == [6, 3]
        eager, captured = engines
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.stepTree(x, x, x, outs[1], masks, nodes=T, sharedMasks=True)
            captured.commitTree(x, x, index, accepted, nodes=T)
        for _ in range(5):                     # 6 + 2 * 5 = 16: eight more still fit
            eager.stepTree(x, x, x, outs[0], masks, nodes=T, sharedMasks=True)
            eager.commitTree(x, x, index, accepted, nodes=T)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(eager.lens, captured.lens) and torch.equal(eager.k, captured.k)
            # (the captured step is planned for another length: the same numbers added up in another order)
            assert ((outs[0] - outs[1]).abs() <= 2.0 ** -10 * outs[0].abs() + 2.0 ** -11).all()
        e.sync()
        for _ in range(6):                     # the first sequence is full after four of them
            graph.replay()
        torch.cuda.synchronize()               # (replays are on torch's stream)
        with pytest.raises(RunntimeError, match="status"):
            e.sync()
        assert captured.lens.tolist() == [24, 14]
        del graph
    finally:
        e.dispose()
