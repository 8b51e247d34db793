"""Batched entry points over the C ABI, for callers that hold many sequences:

- ``prefill_batched``: padded-batch prefill (``batch`` sequences of
  ``seqStride`` rows, per-sequence lengths) — the packed-segments form of the
  reference (packages/runntime/src/zoo/minilm/model.ts:167-185) computed on the
  fly from the lengths.
- ``decode_batched``: one decode step for ``batch`` KV caches with the append
  fused — the step of packages/runntime/src/zoo/moonshine/decoder.ts:58-76 for
  many sequences at once; ``KvCacheEngine`` keeps the caches and lengths like
  the transcriber does (transcriber.ts:111-118,161-203).
- ``PeerExchangeDecode`` / ``ShardedDecode``: long-context decode with the KV
  sequence split across ranks; each rank attends to its rows, the (m, l, acc)
  partials go to the rank that merges the sequence through peer memory, or are
  all-gathered by NCCL, and are merged (algebra of attnDecode.ts:405-422).
  ``ShardedKvCacheEngine`` is the KV-cache engine over caches sharded by position,
  ``ExchangeMemory`` the set-up of the peer buffers through the C ABI.
- a speculative decode step, which answers several drafted tokens of every sequence at
  once: ``rotary_batched`` (q and k turned by integer positions; ``rotary_plan`` makes its
  frequencies), ``tree_batched`` (the tokens attend to the caches and to their ancestors;
  ``tree_masks``), ``verify_batched`` (which of them stand, by the target's probabilities)
  and ``commit_batched`` (their keys and values into the caches).  ``KvCacheEngine`` has
  them as ``stepTree`` / ``stepTreeQkv`` and ``commitTree`` / ``commitTreeQkv``.

Tensors are passed as device pointers (ints) or as anything with
``data_ptr()`` (torch tensors).  torch is used only for device memory and
``torch.distributed``.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple

from ._lib import (AttnArgs, CommitArgs, CommitCountedArgs, DecodeArgs, DecodeSecond, DTYPE_CODE, Exchange, MAX_NODES,
                   MAX_ROTARY_WINDOWS, RotaryArgs, TreeArgs, VerifyArgs, WINDOW_INF, call, check)
from .executor import CudaExecutor


def _ptr(x) -> Optional[int]:
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return int(x.data_ptr())


def _win(w) -> int:
    if w is None or w == float("inf"):
        return WINDOW_INF
    return min(int(w), WINDOW_INF)


def prefill_batched(ex: CudaExecutor, q, k, v, out, *, dtype: str, batch: int, seqStride: int,
                    seqLens, qHeads: int, kvHeads: int, headDim: int, windowLeft=None,
                    windowRight=None, sinks=None) -> None:
    """q/out: [batch*seqStride, qHeads*headDim]; k/v: [batch*seqStride,
    kvHeads*headDim]; seqLens: device int32 [batch].  Row r of sequence b sees
    keys of sequence b only, inside the window, below seqLens[b]; rows at or
    past seqLens[b] come out zero."""
    a = AttnArgs()
    a.q, a.k, a.v, a.out = _ptr(q), _ptr(k), _ptr(v), _ptr(out)
    a.sinks = _ptr(sinks)
    a.dtype = DTYPE_CODE[dtype]
    a.qLen = a.kvLen = batch * seqStride
    a.qHeads, a.kvHeads, a.headDim = qHeads, kvHeads, headDim
    a.windowLeft, a.windowRight = _win(windowLeft), _win(windowRight)
    a.seqStride, a.seqLens = seqStride, _ptr(seqLens)
    check(ex._lib.rt_attn(ex.ctx, C.byref(a)), ex.ctx)


def decode_batched(ex: CudaExecutor, q, out, kCache, vCache, *, dtype: str, batch: int,
                   cacheRows: int, qHeads: int, kvHeads: int, headDim: int, kvLen: int = 0,
                   kvLens=None, kNew=None, vNew=None, cacheSeqStride: Optional[int] = None,
                   windowLeft=None, sinks=None, partialsOut=None, splits: int = 0,
                   ropeCos=None, ropeSin=None, ropeByPosition: bool = False, qRowStride: int = 0,
                   kNewRowStride: int = 0, vNewRowStride: int = 0, exchange=None,
                   kvSharded: bool = False, shardStart: int = 0, kCachePtrs=None, vCachePtrs=None,
                   second=None) -> None:
    """One decode step for ``batch`` sequences; see rt_attn_decode in
    include/rt_attn.h.  ``kvLen`` is the (maximum) visible length including the
    appended row; ``kvLens`` gives it per sequence.  With ``ropeCos``/``ropeSin``
    q and kNew are un-rotated rows (for example windows of the fused qkv
    projection, ``*RowStride`` apart) and the kernel rotates them.
    ``kCachePtrs``/``vCachePtrs``: device int64 arrays [batch] of cache addresses, for
    caches allocated one by one (``kCache``/``vCache`` may then be None).  ``second``
    (from ``second_attention``): a cross-attention computed by the same launch."""
    d = DecodeArgs()
    d.q, d.out = _ptr(q), _ptr(out)
    d.kCache, d.vCache = _ptr(kCache), _ptr(vCache)
    d.kNew, d.vNew = _ptr(kNew), _ptr(vNew)
    d.kvLens, d.sinks, d.partialsOut = _ptr(kvLens), _ptr(sinks), _ptr(partialsOut)
    d.cacheSeqStride = (cacheRows * kvHeads * headDim) if cacheSeqStride is None else cacheSeqStride
    d.dtype = DTYPE_CODE[dtype]
    d.batch, d.cacheRows, d.kvLen = batch, cacheRows, kvLen
    d.qHeads, d.kvHeads, d.headDim = qHeads, kvHeads, headDim
    d.windowLeft, d.splits = _win(windowLeft), splits
    d.ropeCos, d.ropeSin, d.ropeByPosition = _ptr(ropeCos), _ptr(ropeSin), int(ropeByPosition)
    d.qRowStride, d.kNewRowStride, d.vNewRowStride = qRowStride, kNewRowStride, vNewRowStride
    if exchange is not None:
        d.exchange = C.pointer(exchange)
    d.kvSharded, d.shardStart = int(kvSharded), shardStart
    d.kCachePtrs, d.vCachePtrs = _ptr(kCachePtrs), _ptr(vCachePtrs)
    if second is not None:
        d.second = C.pointer(second)
    check(ex._lib.rt_attn_decode(ex.ctx, C.byref(d)), ex.ctx)


def second_attention(q, out, kCache, vCache, *, cacheRows: int, qHeads: int, kvHeads: int,
                     headDim: int, kvLen: int = 0, kvLens=None, windowLeft=None,
                     cacheSeqStride: Optional[int] = None, qRowStride: int = 0, kCachePtrs=None,
                     vCachePtrs=None) -> DecodeSecond:
    """The ``second`` argument of decode_batched: a cross-attention (no append, no rope)
    that shares the launch of a self-attention step — the two attentions of a decoder
    layer (packages/runntime/src/zoo/moonshine/decoder.ts:58-76, 105-109) in one kernel."""
    x = DecodeSecond()
    x.q, x.out = _ptr(q), _ptr(out)
    x.kCache, x.vCache = _ptr(kCache), _ptr(vCache)
    x.kCachePtrs, x.vCachePtrs = _ptr(kCachePtrs), _ptr(vCachePtrs)
    x.kvLens = _ptr(kvLens)
    x.cacheSeqStride = (cacheRows * kvHeads * headDim) if cacheSeqStride is None else cacheSeqStride
    x.qRowStride = qRowStride
    x.cacheRows, x.kvLen, x.windowLeft = cacheRows, (kvLen or cacheRows), _win(windowLeft)
    return x


def merge_partials(ex: CudaExecutor, partials, parts: int, units: int, headDim: int, out,
                   dtype: str) -> None:
    check(ex._lib.rt_attn_merge_partials(ex.ctx, C.c_void_p(_ptr(partials)), parts, units,
                                         headDim, C.c_void_p(_ptr(out)), DTYPE_CODE[dtype]),
          ex.ctx)


class RotaryPlan:
    """Frequencies of rotary_batched on the device: ``rotaryDim`` columns of a head turn, pair i by
    ``turns[i]`` / 2^64 of a whole turn per position, and are multiplied by ``scale``."""

    def __init__(self, rotaryDim: int, turns, scale: float):
        self.rotaryDim, self.turns, self.scale = rotaryDim, turns, scale


def rotary_frequencies(rotaryDim: int, *, base: float = 10000.0,
                       scaling: Optional[dict] = None) -> Tuple[list, float]:
    """(f, scale): the angle per position of every pair, base^(-2i / rotaryDim), and the factor on
    the rotated columns, changed for contexts longer than those trained on by ``scaling``:

    - ``dict(kind="linear", factor=s)``: positions s times as close, f / s;
    - ``dict(kind="base", factor=s)``: a larger base, base * s^(d / (d - 2)), which leaves the
      fastest pair alone and slows the slowest one down s times;
    - ``dict(kind="bands", factor=s, low=a, high=b, original=n)``: by the turns r = n f / (2 pi) that a
      pair makes over the n positions trained on: those below a are slowed down s times, those above
      b are not, f * (g + (1 - g) / s) with g = (r - a) / (b - a) between.

    Each takes ``scale`` too, the factor on the columns (1 by default)."""
    if not isinstance(rotaryDim, int) or rotaryDim < 2 or rotaryDim % 2:
        raise ValueError(f"rotary: rotaryDim {rotaryDim} must be a positive even integer")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"rotary: base {base} must be positive and finite")
    kind = scaling["kind"] if scaling else None
    if kind not in (None, "linear", "base", "bands"):
        raise ValueError(f"rotary: unknown scaling {kind}")
    s = float(scaling["factor"]) if scaling else 1.0
    if not (s > 0 and math.isfinite(s)):
        raise ValueError(f"rotary: factor {s} must be positive and finite")
    scale = float(scaling.get("scale", 1.0)) if scaling else 1.0
    if not math.isfinite(scale):
        raise ValueError(f"rotary: scale {scale} must be finite")
    if kind == "base" and rotaryDim > 2:
        base = base * s ** (rotaryDim / (rotaryDim - 2))
    f = [base ** (-2.0 * i / rotaryDim) for i in range(rotaryDim // 2)]
    if kind == "linear":
        f = [x / s for x in f]
    elif kind == "bands":
        low, high, n = float(scaling["low"]), float(scaling["high"]), scaling["original"]
        if not low < high or not n > 0:
            raise ValueError(f"rotary: bands need low {low} < high {high} and original {n} positive")
        keep = [min(max((n * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        f = [x * (g + (1.0 - g) / s) for x, g in zip(f, keep)]
    return f, scale


def rotary_plan(rotaryDim: int, *, base: float = 10000.0, scaling: Optional[dict] = None,
                device=None) -> RotaryPlan:
    """The plan of rotary_batched for ``rotary_frequencies(rotaryDim, base=base, scaling=scaling)``, on ``device`` (the
    executor's; torch's default device, which is the CPU as a rule, if None)."""
    import torch
    f, scale = rotary_frequencies(rotaryDim, base=base, scaling=scaling)
    turns = [int(x / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for x in f]
    turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device=device)
    return RotaryPlan(rotaryDim, turns, scale)


_HALVES = {"interleaved": 0, "half": 1}


def rotary_batched(ex: CudaExecutor, x, positions, plan: RotaryPlan, windows: Sequence[tuple], *,
                   dtype: str, rows: int, headDim: int, layout: str = "interleaved", xRowStride: int,
                   inverse: bool = False) -> None:
    """Rotary positions by rt_rotary (include/rt_attn.h): the first ``plan.rotaryDim`` columns of the heads in
    ``windows`` of ``x`` (rows ``xRowStride`` elements apart) are turned by ``positions`` (device int32 [rows]).
    A window is ``(first column, heads, out)`` or ``(first column, heads, out, outRowStride)``; ``out`` may be the
    window itself.  ``layout``: pairs of adjacent columns ("interleaved") or of the two halves ("half").
    ``inverse`` turns the other way: with the outputs' gradients in place of x that is the backward pass."""
    if layout not in _HALVES:
        raise ValueError(f"rotary: layout {layout} must be 'interleaved' or 'half'")
    n = len(windows)
    if not 1 <= n <= MAX_ROTARY_WINDOWS:
        raise ValueError(f"rotary: takes 1..{MAX_ROTARY_WINDOWS} windows, got {n}")
    if getattr(plan.turns, "is_cuda", True) is False:
        raise ValueError(f"rotary: the plan is on {plan.turns.device}: rotary_plan's device is the executor's")
    flat = []
    for w in windows:
        flat += (w[0], w[2], w[3] if len(w) > 3 else 0, w[1], 0)
    flat += (0, None, 0, 0, 0) * (MAX_ROTARY_WINDOWS - n)
    # (fields in the order of the structure)
    call(ex._lib, "rt_rotary", ex.ctx, RotaryArgs, x, positions, plan.turns, rows, xRowStride, headDim,
         plan.rotaryDim, _HALVES[layout], 1 if inverse else 0, plan.scale, DTYPE_CODE[dtype], n, *flat)


def tree_masks(parents: Sequence[int]) -> list:
    """The masks of tree_batched for a tree given by its parents (-1: none; a parent comes before its
    children): bit j of mask i is set where node j is node i or an ancestor of it.  As signed 64-bit
    integers, for ``torch.tensor(..., dtype=torch.int64)``."""
    if not 1 <= len(parents) <= MAX_NODES:
        raise ValueError(f"tree_masks: takes 1..{MAX_NODES} nodes, got {len(parents)}")
    masks: list = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"tree_masks: parent {p} of node {i} must be -1 or an earlier node")
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def tree_batched(ex: CudaExecutor, q, out, kCache, vCache, kNew, vNew, masks, *, dtype: str, batch: int,
                 nodes: int, cacheRows: int, qHeads: int, kvHeads: int, headDim: int, kvLen: int = 0,
                 kvLens=None, nodeCounts=None, sharedMasks: bool = False,
                 cacheSeqStride: Optional[int] = None, windowLeft=None, sinks=None, qRowStride: int = 0,
                 kNewRowStride: int = 0, vNewRowStride: int = 0, splits: int = 0) -> None:
    """Attention of ``nodes`` drafted tokens per sequence over its cache and one another; see rt_attn_tree in
    include/rt_attn.h.  ``q``/``out``: [batch*nodes, qHeads*headDim]; ``kNew``/``vNew``: the tokens' own keys and
    values, which stay outside the caches; ``masks``: device int64 [batch, nodes] (or [nodes] with
    ``sharedMasks``), see tree_masks.  ``kvLens`` (device int32 [batch]) are the rows in the caches, ``kvLen`` their
    maximum, or the length of all without them; ``nodeCounts`` the sequences' own numbers of nodes.  A captured call
    keeps the plan for its ``kvLen``."""
    # (fields in the order of the structure)
    call(ex._lib, "rt_attn_tree", ex.ctx, TreeArgs, q, out, kCache, vCache, kNew, vNew, kvLens, nodeCounts, masks, sinks,
         cacheRows * kvHeads * headDim if cacheSeqStride is None else cacheSeqStride, qRowStride, kNewRowStride,
         vNewRowStride, DTYPE_CODE[dtype], batch, nodes, cacheRows, kvLen, qHeads, kvHeads, headDim, _win(windowLeft),
         1 if sharedMasks else 0, splits)


def tree_route(ex: CudaExecutor, *, dtype: str, **sizes) -> str:
    """Which kernel tree_batched runs for these sizes (tensors on 16-byte boundaries, dense)."""
    a = TreeArgs()
    a.q = a.out = a.kCache = a.vCache = a.kNew = a.vNew = a.masks = 16
    a.dtype, a.windowLeft = DTYPE_CODE[dtype], WINDOW_INF
    for name, value in sizes.items():
        setattr(a, name, value)
    a.cacheSeqStride = a.cacheSeqStride or a.cacheRows * a.kvHeads * a.headDim
    route = C.c_char_p()
    check(ex._lib.rt_attn_tree_route(ex.ctx, C.byref(a), C.byref(route)), ex.ctx)
    return route.value.decode()


def verify_batched(ex: CudaExecutor, target, tokens, accept, sample, path, outTokens, accepted, *,
                   dtype: str, batch: int, nodes: int, vocab: int, draft=None, parents=None,
                   nodeCounts=None, targetRowStride: int = 0, targetSeqStride: int = 0,
                   draftRowStride: int = 0, draftSeqStride: int = 0) -> None:
    """Which drafted tokens stand, and the token after them, by rt_verify_drafts (include/rt_attn.h).
    ``target``/``draft``: probabilities [batch, nodes + 1, vocab], row 0 after the text and row i + 1 after node i;
    ``tokens``/``parents``: device int32 [batch, nodes] (``parents`` None: a chain); ``accept`` f32 [batch, nodes] and
    ``sample`` f32 [batch] are uniform in [0, 1).  Written, all int32: ``path`` [batch, nodes], ``outTokens``
    [batch, nodes + 1], ``accepted`` [batch]."""
    call(ex._lib, "rt_verify_drafts", ex.ctx, VerifyArgs, target, draft, tokens, parents, nodeCounts, accept, sample, path,
         outTokens, accepted, targetRowStride, targetSeqStride, draftRowStride, draftSeqStride, DTYPE_CODE[dtype],
         batch, nodes, vocab)


def commit_batched(ex: CudaExecutor, caches: Sequence, fresh: Sequence, index, counts, kvLens, *, dtype: str,
                   batch: int, nodes: int, cacheRows: int, width: int, lead: int = 0,
                   cacheSeqStride: Optional[int] = None, freshRowStride: int = 0,
                   indexStride: int = 0, committed=None) -> None:
    """Rows of the tokens that stand into the caches, by rt_commit_rows (include/rt_attn.h): for every tensor of
    ``caches`` (K and V of all layers, [batch, cacheRows, width] each: a sequence of them or one tensor) rows
    ``kvLens[b]``... become rows 0..lead-1 and lead + ``index[b][j]``, j < ``counts[b]``, of its [batch*nodes, width]
    tensor in ``fresh``.
    ``index`` and ``counts`` are verify_batched's ``path`` and ``accepted``; ``kvLens`` is not advanced.  ``committed``
    (device int32 [batch]) becomes what each sequence's length grows by: 0 for one that was left alone."""
    n = len(caches)
    if n != len(fresh):
        raise ValueError(f"commit: {n} caches and {len(fresh)} tensors of new rows")
    values = (_each(caches), _each(fresh), index, counts, kvLens,
              cacheRows * width if cacheSeqStride is None else cacheSeqStride, freshRowStride, width, DTYPE_CODE[dtype], n,
              batch, nodes, cacheRows, lead, indexStride)
    if committed is None:
        call(ex._lib, "rt_commit_rows", ex.ctx, CommitArgs, *values)
    else:
        call(ex._lib, "rt_commit_rows_counted", ex.ctx, CommitCountedArgs, *values, committed)


def _each(tensors):
    """The addresses of the parts of one tensor along its first dimension; a sequence of tensors as it is (taking a tensor
    apart costs two microseconds for each part)."""
    if not hasattr(tensors, "data_ptr"):
        return tensors
    base, step = tensors.data_ptr(), tensors.stride(0) * tensors.element_size()
    return range(base, base + len(tensors) * step, step) if step else [base] * len(tensors)


def _check_tensor(call: str, name: str, x, kind: str, device, rows: int, cols: int, stride: int) -> None:
    """Refuses a tensor that does not hold what a kernel reads from its address on: ``rows`` times ``cols`` numbers
    of ``kind`` (or, of integers, the unsigned kind), ``stride`` elements from one row to the next.  Addresses are
    taken as they are."""
    if not hasattr(x, "dtype"):
        return
    if x.device != device:
        raise ValueError(f"{call}: {name} is on {x.device}, not on {device}")
    if str(x.dtype) not in ("torch." + kind, "torch.u" + kind):
        raise ValueError(f"{call}: {name} is {x.dtype}, not torch.{kind}")
    if x.is_contiguous() and (x.dim() != 2 or rows == 1 or x.shape[1] == stride):
        fits = cols == 0 or x.numel() >= (rows - 1) * stride + cols
    else:
        fits = cols == 0 or x.dim() == 2 and x.shape[0] >= rows and x.shape[1] >= cols and x.stride() == (stride, 1)
    if not fits:
        raise ValueError(f"{call}: {name} of shape {tuple(x.shape)} and strides {tuple(x.stride())} does not hold {rows} rows "
                         f"of {cols}, {stride} elements apart")


class KvCacheEngine:
    """Preallocated self-attention caches for ``batch`` sequences plus their
    lengths, stepped one token at a time: append + causal attend in one kernel.
    Optionally a fixed cross-attention K/V (encoder states) per sequence.  The
    lengths are advanced by torch and read by the library's kernels, so every
    step binds the executor to torch's current stream first."""

    def __init__(self, ex: CudaExecutor, *, batch: int, maxPositions: int, qHeads: int,
                 kvHeads: int, headDim: int, dtype: str = "f16", windowLeft=None, device=None):
        import torch
        self.ex, self.batch, self.maxPositions = ex, batch, maxPositions
        self.qHeads, self.kvHeads, self.headDim, self.dtype = qHeads, kvHeads, headDim, dtype
        self.windowLeft = windowLeft
        dev = device if device is not None else torch.device("cuda", ex.device)
        tdt = torch.float16 if dtype == "f16" else torch.float32
        kvw = kvHeads * headDim
        self.k = torch.zeros(batch, maxPositions, kvw, dtype=tdt, device=dev)
        self.v = torch.zeros(batch, maxPositions, kvw, dtype=tdt, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.committed = torch.zeros_like(self.lens)      # rows of the last commitTree
        self.maxLen, self.exact = 0, True     # the longest sequence, or a bound of it
        self.cross: Optional[Tuple[object, object, int]] = None
        self.rope = None
        self.rotary = None

    def setCross(self, k, v, rows: int) -> None:
        """Precomputed cross-attention K/V [batch, rows, kvHeads*headDim]."""
        self.cross = (k, v, rows)

    def setRope(self, cos, sin) -> None:
        """Pair-duplicated f32 tables [maxPositions, headDim] (any scale folded in,
        packages/runntime/src/zoo/moonshine/rope.ts:18-50); stepQkv then rotates."""
        self.rope = (cos, sin)

    def stepQkv(self, qkv, out) -> None:
        """One decoder-layer step from the fused projection's rows
        qkv [batch, (qHeads + 2*kvHeads)*headDim] (columns q|k|v, un-rotated): rope
        on q and k at each sequence's position, append, causal attend — the six
        dispatches of packages/runntime/src/zoo/moonshine/decoder.ts:66-76 in one call."""
        qw, kvw = self.qHeads * self.headDim, self.kvHeads * self.headDim
        es = qkv.element_size()
        base = qkv.data_ptr()
        cos, sin = self.rope
        _bind_to_torch_stream(self.ex)
        self._advance()
        decode_batched(self.ex, base, out, self.k, self.v, dtype=self.dtype, batch=self.batch,
                       cacheRows=self.maxPositions, qHeads=self.qHeads, kvHeads=self.kvHeads,
                       headDim=self.headDim, kvLen=self.maxLen, kvLens=self.lens,
                       kNew=base + qw * es, vNew=base + (qw + kvw) * es,
                       windowLeft=self.windowLeft, ropeCos=cos, ropeSin=sin, ropeByPosition=True,
                       qRowStride=qw + 2 * kvw, kNewRowStride=qw + 2 * kvw,
                       vNewRowStride=qw + 2 * kvw)

    def _room(self, rows: int) -> None:
        """``rows`` more have to fit behind the longest sequence.  After commitTree the host knows a bound
        of the lengths alone (how many drafted tokens stood is on the device); where that is too large
        it asks.  Under a capture it cannot: then the kernels alone refuse what has no room, as they do in every replay."""
        if self.maxLen + rows > self.maxPositions and not self.exact and rows <= self.maxPositions:
            if _capturing():
                self.maxLen = self.maxPositions - rows
                return
            self.maxLen, self.exact = int(self.lens.max().item()), True
        if self.maxLen + rows > self.maxPositions:
            raise ValueError(
                f"writeRows: rows [{self.maxLen}, {self.maxLen + rows}) exceed dst capacity "
                f"{self.maxPositions}")

    def _advance(self) -> None:
        self._room(1)
        self.lens.add_(1)
        self.maxLen += 1

    def step(self, q, kNew, vNew, out) -> None:
        """Appends kNew/vNew at each sequence's end and attends causally."""
        _bind_to_torch_stream(self.ex)
        self._advance()
        decode_batched(self.ex, q, out, self.k, self.v, dtype=self.dtype, batch=self.batch,
                       cacheRows=self.maxPositions, qHeads=self.qHeads, kvHeads=self.kvHeads,
                       headDim=self.headDim, kvLen=self.maxLen, kvLens=self.lens, kNew=kNew,
                       vNew=vNew, windowLeft=self.windowLeft)

    def stepWithCross(self, q, kNew, vNew, out, qCross, outCross) -> None:
        """The self-attention step (append + causal attend) and the cross-attention over
        the encoder states set by setCross, in one launch."""
        k, v, rows = self.cross
        _bind_to_torch_stream(self.ex)
        self._advance()
        sec = second_attention(qCross, outCross, k, v, cacheRows=rows, qHeads=self.qHeads,
                               kvHeads=self.kvHeads, headDim=self.headDim, kvLen=rows)
        decode_batched(self.ex, q, out, self.k, self.v, dtype=self.dtype, batch=self.batch,
                       cacheRows=self.maxPositions, qHeads=self.qHeads, kvHeads=self.kvHeads,
                       headDim=self.headDim, kvLen=self.maxLen, kvLens=self.lens, kNew=kNew,
                       vNew=vNew, windowLeft=self.windowLeft, second=sec)

    def _check_qkv(self, call: str, qkv, nodes: int) -> None:
        width = (self.qHeads + 2 * self.kvHeads) * self.headDim
        _check_tensor(call, "qkv", qkv, "float16" if self.dtype == "f16" else "float32", self.lens.device, self.batch * nodes,
                      width, width)

    def setRotary(self, plan: RotaryPlan, layout: str = "interleaved") -> None:
        """Frequencies of stepTreeQkv's rotary positions."""
        self.rotary = (plan, layout)

    def stepTree(self, q, kNew, vNew, out, masks, *, nodes: int, nodeCounts=None, sharedMasks: bool = False,
                 qRowStride: int = 0, kNewRowStride: int = 0, vNewRowStride: int = 0, sinks=None) -> None:
        """``nodes`` drafted tokens of every sequence attend to its cache and to their ancestors
        (tree_batched).  Nothing is appended: commitTree does that for the tokens that stand.  A captured step keeps the
        plan of the lengths at its capture: replayed with caches many times as long it is right, but slower than a step captured at
        such lengths (or a tree_batched with kvLen = cacheRows)."""
        device = self.lens.device
        _check_tensor("stepTree", "masks", masks, "int64", device, 1 if sharedMasks else self.batch, nodes, nodes)
        _check_tensor("stepTree", "nodeCounts", nodeCounts, "int32", device, 1, self.batch, self.batch)
        _check_tensor("stepTree", "sinks", sinks, "float32", device, 1, self.qHeads, self.qHeads)
        _bind_to_torch_stream(self.ex)
        self._room(nodes)
        tree_batched(self.ex, q, out, self.k, self.v, kNew, vNew, masks, dtype=self.dtype, batch=self.batch,
                     nodes=nodes, cacheRows=self.maxPositions, qHeads=self.qHeads, kvHeads=self.kvHeads,
                     headDim=self.headDim, kvLen=self.maxLen, kvLens=self.lens, nodeCounts=nodeCounts,
                     sharedMasks=sharedMasks, windowLeft=self.windowLeft, sinks=sinks, qRowStride=qRowStride,
                     kNewRowStride=kNewRowStride, vNewRowStride=vNewRowStride)

    def stepTreeQkv(self, qkv, out, masks, depths, *, nodes: int, nodeCounts=None, sharedMasks: bool = False,
                    sinks=None) -> None:
        """stepTree from the fused projection's rows qkv [batch*nodes, (qHeads + 2*kvHeads)*headDim] (columns
        q|k|v): q and k are turned in place by setRotary's plan at the sequence's length plus ``depths``
        (device int32 [nodes] or [batch, nodes]).  qkv then holds the keys and values that
        commitTreeQkv takes."""
        if self.rotary is None:
            raise ValueError("stepTreeQkv: setRotary has not been called")
        plan, layout = self.rotary
        if depths.dtype != self.lens.dtype:
            raise ValueError(f"stepTreeQkv: depths are {depths.dtype}, not {self.lens.dtype}")
        if tuple(depths.shape) not in ((nodes,), (1, nodes), (self.batch, nodes)):
            raise ValueError(f"stepTreeQkv: depths of shape {tuple(depths.shape)} are neither [{nodes}] nor "
                             f"[{self.batch}, {nodes}]")
        qw, kvw = self.qHeads * self.headDim, self.kvHeads * self.headDim
        width, es, base = qw + 2 * kvw, qkv.element_size(), qkv.data_ptr()
        self._check_qkv("stepTreeQkv", qkv, nodes)
        _bind_to_torch_stream(self.ex)
        self._room(nodes)
        positions = (self.lens[:, None] + depths).contiguous()   # (a sum has its operands' order in memory)
        rotary_batched(self.ex, base, positions, plan,
                       [(0, self.qHeads, base, width), (qw, self.kvHeads, base + qw * es, width)], dtype=self.dtype,
                       rows=self.batch * nodes, headDim=self.headDim, layout=layout, xRowStride=width)
        self.stepTree(base, base + qw * es, base + (qw + kvw) * es, out, masks, nodes=nodes, nodeCounts=nodeCounts,
                      sharedMasks=sharedMasks, qRowStride=width, kNewRowStride=width, vNewRowStride=width,
                      sinks=sinks)

    def commitTree(self, kNew, vNew, index, accepted, *, nodes: int, lead: int = 1, freshRowStride: int = 0,
                   indexStride: int = 0) -> None:
        """Keys and values of the first ``lead`` nodes and of those in ``index`` (verify_batched's ``path`` and
        ``accepted``) go to the ends of the caches, and the lengths grow by them.  With lead = 1 node 0 is the
        token that the last step ended with and the others are the verified ones, nodes - 1 to a row of
        ``index`` unless indexStride says otherwise.  Every sequence gets its ``lead`` rows; where some have
        ended, lead = 0 with all of a sequence's rows in ``index``, none of an ended one.  A sequence whose rows do
        not fit or whose indices are out of range is left as it is, its length too (``committed`` 0), and the
        executor's sync reports it."""
        stride = indexStride or max(nodes - lead, 1)
        device = self.lens.device
        _check_tensor("commitTree", "accepted", accepted, "int32", device, 1, self.batch, self.batch)
        _check_tensor("commitTree", "index", index, "int32", device, self.batch, max(nodes - lead, 0), stride)
        _bind_to_torch_stream(self.ex)
        commit_batched(self.ex, (self.k, self.v), (kNew, vNew), index, accepted, self.lens, dtype=self.dtype,
                       batch=self.batch, nodes=nodes, cacheRows=self.maxPositions,
                       width=self.kvHeads * self.headDim, lead=lead, freshRowStride=freshRowStride,
                       indexStride=stride, committed=self.committed)
        self.lens.add_(self.committed)
        self.maxLen, self.exact = min(self.maxLen + nodes, self.maxPositions), False

    def commitTreeQkv(self, qkv, index, accepted, *, nodes: int, lead: int = 1, indexStride: int = 0) -> None:
        """commitTree from the rows that stepTreeQkv has turned."""
        qw, kvw = self.qHeads * self.headDim, self.kvHeads * self.headDim
        self._check_qkv("commitTreeQkv", qkv, nodes)
        es, base = qkv.element_size(), qkv.data_ptr()
        self.commitTree(base + qw * es, base + (qw + kvw) * es, index, accepted, nodes=nodes, lead=lead,
                        freshRowStride=qw + 2 * kvw, indexStride=indexStride)

    def crossAttend(self, q, out) -> None:
        k, v, rows = self.cross
        _bind_to_torch_stream(self.ex)
        decode_batched(self.ex, q, out, k, v, dtype=self.dtype, batch=self.batch, cacheRows=rows,
                       qHeads=self.qHeads, kvHeads=self.kvHeads, headDim=self.headDim, kvLen=rows)


def shard_rows(total: int, world: int, rank: int) -> Tuple[int, int]:
    """Rows [start, end) of a ``total``-row KV sequence that live on ``rank``:
    contiguous, balanced to within one row."""
    base, extra = divmod(total, world)
    start = rank * base + min(rank, extra)
    return start, start + base + (1 if rank < extra else 0)


def shard_of_position(position: int, shardRows: int) -> Tuple[int, int]:
    """(rank, local row) of a token position when every rank's cache holds
    ``shardRows`` consecutive positions: position t lives on rank t // shardRows."""
    return position // shardRows, position % shardRows


def owned_sequences(batch: int, world: int, rank: int) -> Tuple[int, int]:
    """(first, count) of the sequences whose partials ``rank`` merges in the cross-GPU
    exchange: contiguous blocks balanced to within one sequence (batch >= world, so
    every rank owns at least one)."""
    first, end = shard_rows(batch, world, rank)
    return first, end - first


def exchange_sizes(world: int, batch: int, qHeads: int, headDim: int) -> Tuple[int, int, int]:
    """(floats of a rank's exchange buffer, 32-bit words of its control block, floats of
    its staging buffer): two halves of [world, per * qHeads, 2+headDim] partials for the
    ``per`` sequences it owns; [world] arrival words + [world + 3] counters; the rank's own
    [batch * qHeads, 2+headDim] rows before they go to their owners."""
    per = -(-batch // world)
    row = 2 + headDim
    return 2 * world * per * qHeads * row, 2 * world + 3, batch * qHeads * row


def make_exchange(world: int, rank: int, partialPtrs, controlPtrs, stagePtr) -> Exchange:
    """rt_exchange over every rank's exchange buffer and control block as mapped in
    this process (``controlPtrs[r]``: rank r's [world] arrival words, then its counters,
    all zero at the start) and this rank's staging buffer."""
    x = Exchange()
    x.world, x.rank = world, rank
    for r in range(world):
        x.partials[r] = _ptr(partialPtrs[r])
        x.flags[r] = _ptr(controlPtrs[r])
    x.step = _ptr(controlPtrs[rank]) + 4 * world
    x.stage = _ptr(stagePtr)
    return x


class ExchangeMemory:
    """A rank's exchange block allocated and mapped through the C ABI (rt_xmem_*):
    what a host without torch.distributed uses.  Processes trade ``export()`` handles
    (64 bytes) and ``importHandle`` them; ranks living in one process ``attach`` each
    other's objects."""

    def __init__(self, device: int, world: int, rank: int, batch: int, qHeads: int,
                 headDim: int):
        from . import _lib
        self._lib = _lib.load()
        h = C.c_void_p()
        check(self._lib.rt_xmem_create(device, world, rank, batch, qHeads, headDim, C.byref(h)))
        self._h, self.world, self.rank = h, world, rank

    def export(self) -> bytes:
        from ._lib import XMEM_HANDLE_BYTES
        buf = C.create_string_buffer(XMEM_HANDLE_BYTES)
        check(self._lib.rt_xmem_export(self._h, buf))
        return buf.raw

    def importHandle(self, peer: int, handle: bytes) -> None:
        check(self._lib.rt_xmem_import(self._h, peer, C.create_string_buffer(handle, len(handle))))

    def attach(self, peer: int, other: "ExchangeMemory") -> None:
        check(self._lib.rt_xmem_attach(self._h, peer, other._h))

    def exchange(self) -> Exchange:
        x = Exchange()
        check(self._lib.rt_xmem_exchange(self._h, C.byref(x)))
        return x

    def destroy(self) -> None:
        if self._h is not None:
            check(self._lib.rt_xmem_destroy(self._h))
            self._h = None


def _bind_to_torch_stream(ex: CudaExecutor) -> None:
    """Engines mix torch work (length updates, collectives) with the library's kernels: both must be on
    one stream, so they put the executor on torch's current stream of its device before every step (a
    context's own stream is non-blocking and would not be ordered with torch's).  The stream's handle
    alone where torch gives it: a stream object takes 3.7 us to make."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    ex.setStream(raw(ex.device) if raw is not None else torch.cuda.current_stream(ex.device).cuda_stream)


def _capturing() -> bool:
    import torch
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


class PeerExchangeDecode:
    """KV-sequence-sharded decode whose ranks trade partials through peer memory:
    the decode kernel sends each sequence's (m, l, acc) rows to the rank that owns the
    sequence and signals it; that rank's merge kernel waits for all ranks' rows of the
    step and merges — no library collective on the step.  ``out`` receives the rows of
    this rank's own sequences (``self.first``, ``self.owned``).  One process per GPU;
    the buffers come from torch's symmetric memory (``transport="symm"``) or from the
    library's own CUDA-IPC set-up (``transport="ipc"``, handles carried by
    ``all_gather_object``).  Kernels run on torch's current stream."""

    def __init__(self, *, batch: int, qHeads: int, headDim: int, device, group=None,
                 transport: str = "symm"):
        import os
        import torch
        import torch.distributed as dist
        self.world = dist.get_world_size(group)
        self.rank = dist.get_rank(group)
        self.first, self.owned = owned_sequences(batch, self.world, self.rank)
        self.transport = transport
        if transport == "ipc":
            index = device.index if device.index is not None else torch.cuda.current_device()
            self.mem = ExchangeMemory(index, self.world, self.rank, batch, qHeads, headDim)
            handles = [None] * self.world
            dist.all_gather_object(handles, self.mem.export(), group=group)
            for r, h in enumerate(handles):
                if r != self.rank:
                    self.mem.importHandle(r, h)
            self.exchange = self.mem.exchange()
            dist.barrier(group)       # every block is mapped (and zero) before anybody signals
            return
        # plain peer mappings only: no NVLink multicast object is bound to these buffers
        os.environ.setdefault("TORCH_SYMM_MEM_DISABLE_MULTICAST", "1")
        import torch.distributed._symmetric_memory as symm
        nfloat, nword, nstage = exchange_sizes(self.world, batch, qHeads, headDim)
        group_name = (group or dist.group.WORLD).group_name
        self.partials = symm.empty(nfloat, dtype=torch.float32, device=device)
        self.control = symm.empty(nword, dtype=torch.int32, device=device)
        self.stage = torch.zeros(nstage, dtype=torch.float32, device=device)
        self.partials.zero_()
        self.control.zero_()
        hp = symm.rendezvous(self.partials, group_name)
        hc = symm.rendezvous(self.control, group_name)
        torch.cuda.synchronize(device)
        dist.barrier(group)           # everybody's words are zero before anybody signals
        self.exchange = make_exchange(self.world, self.rank, [int(p) for p in hp.buffer_ptrs],
                                      [int(p) for p in hc.buffer_ptrs], self.stage)
        self._handles = (hp, hc)

    def step(self, ex: CudaExecutor, q, kShard, vShard, out, *, dtype: str, batch: int,
             shardRows: int, qHeads: int, kvHeads: int, headDim: int, kvLens=None,
             kvLen: Optional[int] = None, kNew=None, vNew=None, shardStart: Optional[int] = None,
             splits: int = 0):
        """One step over this rank's rows.  Without ``shardStart`` the shard is a static
        slab of ``shardRows`` visible rows (``kvLens``: local lengths).  With it the caches
        are sharded by position — this rank holds global rows [shardStart, shardStart +
        shardRows) — ``kvLen``/``kvLens`` are global lengths and ``kNew``/``vNew`` are
        appended by the rank that owns the new position."""
        _bind_to_torch_stream(ex)
        sharded = shardStart is not None
        decode_batched(ex, q, out, kShard, vShard, dtype=dtype, batch=batch, cacheRows=shardRows,
                       qHeads=qHeads, kvHeads=kvHeads, headDim=headDim,
                       kvLen=(kvLen if kvLen is not None else shardRows), kvLens=kvLens,
                       kNew=kNew, vNew=vNew, splits=splits, exchange=self.exchange,
                       kvSharded=sharded, shardStart=shardStart or 0)
        return out


class ShardedKvCacheEngine:
    """The KV-cache engine with every sequence's cache split by position over the ranks
    of an exchange: rank r keeps positions [r*shardRows, (r+1)*shardRows) of all
    ``batch`` sequences (shardRows = ceil(maxPositions / world)).  A step appends the
    new token's K/V row on the rank that owns its position — the others attend without
    it — and merges the ranks' partials; ``out`` receives this rank's own sequences.
    The decoder loop it serves: packages/runntime/src/zoo/moonshine/transcriber.ts:
    111-118,161-203 (caches preallocated per layer, one writeRows + attention per step).
    Kernels run on torch's current stream."""

    def __init__(self, ex: CudaExecutor, exchange: Exchange, *, batch: int, maxPositions: int,
                 qHeads: int, kvHeads: int, headDim: int, dtype: str = "f16", device=None):
        import torch
        self.ex, self.exchange, self.batch = ex, exchange, batch
        self.world, self.rank = exchange.world, exchange.rank
        self.maxPositions = maxPositions
        self.shardRows = -(-maxPositions // self.world)
        self.shardStart = self.rank * self.shardRows
        self.qHeads, self.kvHeads, self.headDim, self.dtype = qHeads, kvHeads, headDim, dtype
        dev = device if device is not None else torch.device("cuda", ex.device)
        tdt = torch.float16 if dtype == "f16" else torch.float32
        kvw = kvHeads * headDim
        self.k = torch.zeros(batch, self.shardRows, kvw, dtype=tdt, device=dev)
        self.v = torch.zeros(batch, self.shardRows, kvw, dtype=tdt, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)   # global lengths
        self.maxLen = 0
        self.first, self.owned = owned_sequences(batch, self.world, self.rank)

    def step(self, q, kNew, vNew, out, *, phases: int = 0) -> None:
        """Appends kNew/vNew [batch, kvHeads*headDim] at each sequence's end (on the rank
        that owns that position) and attends causally over all ranks' rows."""
        _bind_to_torch_stream(self.ex)
        if phases in (0, 1, 3):
            if self.maxLen + 1 > self.maxPositions:
                raise ValueError(
                    f"writeRows: rows [{self.maxLen}, {self.maxLen + 1}) exceed dst capacity "
                    f"{self.maxPositions}")
            self.lens.add_(1)
            self.maxLen += 1
        self.exchange.phases = phases
        decode_batched(self.ex, q, out, self.k, self.v, dtype=self.dtype, batch=self.batch,
                       cacheRows=self.shardRows, qHeads=self.qHeads, kvHeads=self.kvHeads,
                       headDim=self.headDim, kvLen=self.maxLen, kvLens=self.lens, kNew=kNew,
                       vNew=vNew, exchange=self.exchange, kvSharded=True,
                       shardStart=self.shardStart)


class ShardedDecode:
    """KV-sequence-sharded decode.  ``partial_fn(out_partials)`` computes this
    rank's (m, l, acc) partials into a [units, 2+hd] f32 tensor; ``merge_fn
    (gathered, out)`` merges [world, units, 2+hd].  The exchange is one
    all-gather of ``units * (2+hd)`` floats per rank.  The library's kernels and
    the collective run on torch's current stream."""

    def __init__(self, group=None):
        import torch.distributed as dist
        self.dist = dist
        self.group = group
        self.world = dist.get_world_size(group) if dist.is_initialized() else 1
        self.rank = dist.get_rank(group) if dist.is_initialized() else 0
        self._gathered = None

    def gather(self, partials):
        """All-gathers the ranks' partial tensors into [world, units, 2+hd]."""
        import torch
        if self._gathered is None or self._gathered.shape[1:] != partials.shape \
                or self._gathered.device != partials.device:
            self._gathered = torch.empty((self.world, *partials.shape), dtype=partials.dtype,
                                         device=partials.device)
        if self.world == 1:
            self._gathered[0].copy_(partials)
        else:
            # concatenation along dim 0 is the layout every backend accepts
            flat = self._gathered.view(self.world * partials.shape[0], *partials.shape[1:])
            self.dist.all_gather_into_tensor(flat, partials.contiguous(), group=self.group)
        return self._gathered

    def step(self, ex: CudaExecutor, q, kShard, vShard, out, *, dtype: str, batch: int,
             shardRows: int, qHeads: int, kvHeads: int, headDim: int, partials, kvLens=None,
             kvLen: Optional[int] = None, kNew=None, vNew=None, shardStart: Optional[int] = None,
             splits: int = 0):
        """Attends to this rank's rows, exchanges partials, merges into ``out`` (every
        rank gets every sequence).  ``shardStart``/``kvLen``/``kNew``/``vNew``: the
        position-sharded form with append, as in PeerExchangeDecode.step."""
        _bind_to_torch_stream(ex)
        sharded = shardStart is not None
        decode_batched(ex, q, None, kShard, vShard, dtype=dtype, batch=batch,
                       cacheRows=shardRows, qHeads=qHeads, kvHeads=kvHeads, headDim=headDim,
                       kvLen=(kvLen if kvLen is not None else shardRows), kvLens=kvLens, kNew=kNew,
                       vNew=vNew, partialsOut=partials, splits=splits, kvSharded=sharded,
                       shardStart=shardStart or 0)
        gathered = self.gather(partials)
        merge_partials(ex, gathered, self.world, batch * qHeads, headDim, out, dtype)
        return out
