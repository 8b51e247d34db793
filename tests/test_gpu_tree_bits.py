"""How many bits of a probability tree attention keeps, where the scores are exact: what is left is the
result's own rounding and that of 32-bit arithmetic."""
import math

import pytest

from gpu_harness import ex  # noqa: F401
from test_gpu_speculate import Tree, gen, on_torch  # noqa: F401

pytestmark = pytest.mark.gpu


def exact_scores(t):
    """Queries and keys on coarse grids, eight columns of a query not zero: every score is a multiple of 1/8 below 8 in
    size, exact in 32 bits in any order of its sum."""
    torch = t.torch
    g = gen(77)

    def grid(x, steps):
        x.copy_(torch.randint(-steps, steps + 1, x.shape, generator=g, device="cuda").to(x.dtype) / steps)

    for x in (t.k, t.kNew):
        grid(x, 4)
    grid(t.q, 2)
    keep = torch.zeros(t.hd, device="cuda", dtype=torch.bool)
    keep[torch.randperm(t.hd, generator=g, device="cuda")[:8]] = True
    q = t.q[:, :t.heads * t.hd].view(-1, t.heads, t.hd)
    q.masked_fill_(~keep, 0)


def check(t, got):
    """Every element within what the arithmetic may do; returns the largest error over the bound."""
    torch = t.torch
    T, H, K, D, G = t.nodes, t.heads, t.kvHeads, t.hd, t.heads // t.kvHeads
    worst = 0.0
    for b in range(t.B):
        L, n = t.lens[b], t.counts[b]
        mine = got.view(t.B, T, H, D)[b, :n].double()
        seen = torch.tensor(t.seen[b][:n, :n], device="cuda")
        depth = (seen.sum(-1) - 1).clamp(min=0)
        past = torch.ones(n, L, dtype=torch.bool, device="cuda")
        if t.window is not None:
            past &= torch.arange(L, device="cuda") >= (L + depth - t.window)[:, None]
            seen = seen & (depth[:, None] - depth[None] <= t.window)
        mask = torch.cat([past, seen], 1)
        rows = slice(b * T, b * T + n)
        for g in range(K):
            cols = slice(g * D, (g + 1) * D)
            k = torch.cat([t.k[b, :L, cols], t.kNew[rows, cols]]).double()
            v = torch.cat([t.v[b, :L, cols], t.vNew[rows, cols]]).double()
            q = t.q[rows, :H * D].view(n, H, D)[:, g * G:(g + 1) * G].double()
            s = torch.einsum("ngd,kd->ngk", q, k).masked_fill(~mask[:, None], -math.inf)
            top = s.amax(-1, keepdim=True)        # (a node sees itself)
            sink = torch.full_like(top, -math.inf)
            if t.sinks is not None:      # (in the log2 domain)
                sink = (t.sinks[g * G:(g + 1) * G].double() * math.log(2))[None, :, None].expand_as(top)
                top = torch.maximum(top, sink)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True) + torch.exp(sink - top)
            p = p / total
            want, size = torch.einsum("ngk,kd->ngd", p, v), torch.einsum("ngk,kd->ngd", p, v.abs())
            # A weight, relative: log2(e) in 32 bits times a score below 8 (2^-21), the exponent's argument below 64 (half
            # a unit of 2^-18), the exponential and the two halves (2^-22 each): 2^-18 together.  Sums over
            # the keys: the tensor core cuts off, 16 keys at a time, the two halves one after the other, and the 32-bit sum of the
            # weights has fewer additions than that: (keys / 8 + 8) times 2^-22.  Both for numerator and denominator.
            # A weight below 2^-24 of a half's range is held to 2^-33 of the row's largest.
            keys = L + n
            relative = 2 * (2.0 ** -18 + (keys / 8 + 8) * 2.0 ** -22)
            bound = 2.0 ** -11 * want.abs() + relative * size + keys * 2.0 ** -33 * v.abs().max() + 2.0 ** -25
            err = (mine[:, g * G:(g + 1) * G] - want).abs()
            worst = max(worst, float((err / bound).max()))
            assert (err <= bound).all(), (b, g, float((err / bound).max()), float(err.max()))
    return worst


@pytest.mark.parametrize("shape", [(8, 2, 128), (4, 4, 64), (8, 8, 52), (6, 6, 36), (16, 1, 128)])
@pytest.mark.parametrize("window,sinks,splits", [(None, False, 0), (None, True, 5), (20, True, 0)])
def test_tree_keeps_the_bits_of_a_probability(on_torch, shape, window, sinks, splits):
    """Values of either sign: where they cancel, the result's own rounding is small and a weight's error is seen."""
    t = Tree("f16", *shape, 16, [0, 3, 14, 70, 300], window=window, sinks=sinks, seed=4)
    exact_scores(t)
    got = t.call(on_torch, splits=splits)
    on_torch.sync()
    check(t, got)


@pytest.mark.parametrize("shape", [(8, 2, 128), (8, 8, 52)])
@pytest.mark.parametrize("splits", [1, 0])
def test_tree_small_probabilities_add_up(on_torch, shape, splits):
    """A sink, or one key, that outweighs each of 9000 others 2^26 times: together they still weigh something."""
    torch = Tree("f16", *shape, 2, [1]).torch
    t = Tree("f16", *shape, 4, [9001, 300], sinks=True, seed=6)
    t.q.zero_()
    t.v.copy_(t.v.abs())
    t.sinks.fill_(26.37)
    got = t.call(on_torch, splits=splits)
    on_torch.sync()
    check(t, got)
    # the key: the first cache row, whose value is zero
    t.sinks = None
    t.q.fill_(1.0)
    for x in (t.k, t.kNew):
        x.zero_()
    t.k.view(t.B, t.rows, t.kvHeads, t.hd)[:, 0, :, :7] = 2.625        # a score of 18.375, 26.5 binary orders
    t.v[:, 0] = 0
    got = t.call(on_torch, splits=splits)
    on_torch.sync()
    check(t, got)
    assert (got.view(t.B, -1)[0] > 0).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape", [(8, 2, 128), (4, 4, 64), (8, 8, 52), (4, 2, 33)])
@pytest.mark.parametrize("nodes,window,splits", [(1, None, 0), (5, None, 0), (64, None, 0), (5, 100, 0), (17, None, 7), (5, 64, 3)])
def test_tree_meets_every_key_once(on_torch, dtype, shape, nodes, window, splits):
    """Equal scores, and values that are one in one column: a result says how many of the keys of that column were
    met, of how many in all."""
    H, K, D = shape
    t = Tree(dtype, *shape, nodes, [0, 1, 63, 64, 65, 127, 128, 129, 300, 515, 1000], window=window, seed=nodes)
    torch, T, B = t.torch, nodes, t.B
    t.q.zero_()
    t.v.zero_()
    t.vNew.zero_()
    j = torch.arange(t.rows, device="cuda")
    t.v.view(B, t.rows, K, D)[:, j, :, j % D] = 1
    i = torch.arange(T, device="cuda")
    for b in range(B):
        t.vNew.view(B, T, K, D)[b, i, :, (t.lens[b] + i) % D] = 1
    got = t.call(on_torch, splits=splits).view(B, T, H, D).double()
    on_torch.sync()
    half = torch.finfo(t.td).eps / 2
    for b, L in enumerate(t.lens):
        seen = torch.tensor(t.seen[b], device="cuda")
        depth = (seen.sum(-1) - 1).clamp(min=0)
        past = torch.ones(T, L, dtype=torch.bool, device="cuda")
        if window is not None:
            past &= torch.arange(L, device="cuda") >= (L + depth - window)[:, None]
            seen = seen & (depth[:, None] - depth[None] <= window)
        mask = torch.cat([past, seen], 1).double()
        column = torch.nn.functional.one_hot(torch.arange(L + T, device="cuda") % D, D).double()
        want = (mask @ column / mask.sum(-1, keepdim=True))[:, None]
        # Weights are powers of two and their sums whole numbers below 2^24: exact, but for the reciprocal and the product with it
        # (2^-23 each), once for every one of up to 64 parts; and the result's own rounding.  A key more or less is 1/1064.
        assert ((got[b] - want).abs() <= (half + 66 * 2.0 ** -23) * want + 2.0 ** -25).all(), b
