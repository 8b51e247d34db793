"""ctypes binding of librt_attn.so — the same C ABI a Node N-API addon binds.

There is no CPU fallback: if the library is missing the import of anything that
computes fails with NOT_INITIALIZED and says how to build it.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional

from .errors import RunntimeError, code_of_status

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "librt_attn.so")

RT_F32, RT_F16 = 0, 1
WINDOW_INF = 0x3FFFFFFF
OPT_PREFILL_TC = 1
OPT_WAIT_POLLS = 2
XMEM_HANDLE_BYTES = 64
DTYPE_CODE = {"f32": RT_F32, "f16": RT_F16}


class AttnArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("out", C.c_void_p),
        ("sinks", C.c_void_p), ("segments", C.c_void_p),
        ("dtype", C.c_int32), ("qkvPacked", C.c_int32),
        ("qLen", C.c_int64), ("kvLen", C.c_int64),
        ("qHeads", C.c_int32), ("kvHeads", C.c_int32), ("headDim", C.c_int32),
        ("windowLeft", C.c_int32), ("windowRight", C.c_int32), ("maxSegment", C.c_int32),
        ("qPosOffset", C.c_int64),
        ("hasKeyBias", C.c_int32), ("biasStart", C.c_int32), ("biasEnd", C.c_int32),
        ("biasValue", C.c_float),
        ("seqStride", C.c_int32), ("seqLens", C.c_void_p),
    ]


MAX_PEERS = 8


class Exchange(C.Structure):
    """rt_exchange: where the ranks sharing a set of sequences trade partials."""
    _fields_ = [
        ("world", C.c_int32), ("rank", C.c_int32),
        ("partials", C.c_void_p * MAX_PEERS), ("flags", C.c_void_p * MAX_PEERS),
        ("step", C.c_void_p), ("stage", C.c_void_p), ("phases", C.c_int32),
    ]


class DecodeSecond(C.Structure):
    """rt_decode_second: a second attention (cross-attention) in the same decode launch."""
    _fields_ = [
        ("q", C.c_void_p), ("out", C.c_void_p), ("kCache", C.c_void_p), ("vCache", C.c_void_p),
        ("kCachePtrs", C.c_void_p), ("vCachePtrs", C.c_void_p), ("kvLens", C.c_void_p),
        ("cacheSeqStride", C.c_int64), ("qRowStride", C.c_int64),
        ("cacheRows", C.c_int32), ("kvLen", C.c_int32), ("windowLeft", C.c_int32),
    ]


class DecodeArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("out", C.c_void_p), ("kCache", C.c_void_p), ("vCache", C.c_void_p),
        ("kNew", C.c_void_p), ("vNew", C.c_void_p), ("kvLens", C.c_void_p),
        ("sinks", C.c_void_p), ("partialsOut", C.c_void_p),
        ("cacheSeqStride", C.c_int64),
        ("dtype", C.c_int32), ("batch", C.c_int32), ("cacheRows", C.c_int32),
        ("kvLen", C.c_int32), ("qHeads", C.c_int32), ("kvHeads", C.c_int32),
        ("headDim", C.c_int32), ("windowLeft", C.c_int32), ("splits", C.c_int32),
        ("ropeByPosition", C.c_int32), ("ropeCos", C.c_void_p), ("ropeSin", C.c_void_p),
        ("qRowStride", C.c_int64), ("kNewRowStride", C.c_int64), ("vNewRowStride", C.c_int64),
        ("exchange", C.POINTER(Exchange)),
        ("kvSharded", C.c_int32), ("shardStart", C.c_int32),
        ("kCachePtrs", C.c_void_p), ("vCachePtrs", C.c_void_p),
        ("second", C.POINTER(DecodeSecond)),
    ]


class Window(C.Structure):
    """rt_window: a column window, rotated or cut out."""
    _fields_ = [
        ("x", C.c_void_p), ("cosT", C.c_void_p), ("sinT", C.c_void_p), ("out", C.c_void_p),
        ("rows", C.c_int64), ("cols", C.c_int64), ("start", C.c_int64), ("width", C.c_int64),
        ("headDim", C.c_int32),
    ]


MAX_NODES = 64
MAX_ROTARY_WINDOWS = 4


def _struct(name: str, doc: str, fields: str):
    """A structure whose fields are ``type:names`` words: P an address, A an array of addresses, i and q 32- and
    64-bit integers, f a float; and its layout, a letter for each field (csrc/host.cpp's ``call``)."""
    types = {"P": C.c_void_p, "A": C.POINTER(C.c_void_p), "i": C.c_int32, "q": C.c_int64, "f": C.c_float}
    pairs = [(n, w[0]) for w in fields.split() for n in w[2:].split(",")]
    return type(name, (C.Structure,), {"__doc__": doc, "_fields_": [(n, types[t]) for n, t in pairs],
                                       "layout": "".join(t for _, t in pairs)})


# (a rotary window's five fields come MAX_ROTARY_WINDOWS times)
RotaryArgs = _struct("RotaryArgs", "rt_rotary_args, its windows' fields one after the other.",
                     "P:x,positions,turns q:rows,xRowStride i:headDim,rotaryDim,halves,inverse f:scale "
                     "i:dtype,windowCount " +
                     " ".join(f"q:start{w} P:out{w} q:outRowStride{w} i:heads{w},reserved{w}"
                              for w in range(MAX_ROTARY_WINDOWS)))
TreeArgs = _struct("TreeArgs", "rt_tree_args.",
                   "P:q,out,kCache,vCache,kNew,vNew,kvLens,nodeCounts,masks,sinks "
                   "q:cacheSeqStride,qRowStride,kNewRowStride,vNewRowStride "
                   "i:dtype,batch,nodes,cacheRows,kvLen,qHeads,kvHeads,headDim,windowLeft,sharedMasks,splits")
VerifyArgs = _struct("VerifyArgs", "rt_verify_args.",
                     "P:target,draft,tokens,parents,nodeCounts,accept,sample,path,outTokens,accepted "
                     "q:targetRowStride,targetSeqStride,draftRowStride,draftSeqStride i:dtype,batch,nodes,vocab")
CommitArgs = _struct("CommitArgs", "rt_commit_args.",
                     "A:caches,fresh P:index,counts,kvLens q:cacheSeqStride,freshRowStride,width "
                     "i:dtype,tensors,batch,nodes,cacheRows,lead,indexStride")
CommitCountedArgs = _struct("CommitCountedArgs", "rt_commit_counted_args, rt_commit_args' fields first.",
                            "A:caches,fresh P:index,counts,kvLens q:cacheSeqStride,freshRowStride,width "
                            "i:dtype,tensors,batch,nodes,cacheRows,lead,indexStride P:committed")


# name -> (restype, argtypes); every symbol include/rt_attn.h declares.
SYMBOLS = {
    "rt_ctx_create": (C.c_int, [C.c_int, C.POINTER(C.c_void_p)]),
    "rt_ctx_destroy": (C.c_int, [C.c_void_p]),
    "rt_ctx_set_stream": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int]),
    "rt_ctx_set_option": (C.c_int, [C.c_void_p, C.c_int, C.c_int]),
    "rt_last_error": (C.c_char_p, [C.c_void_p]),
    "rt_sync": (C.c_int, [C.c_void_p]),
    "rt_launch_count": (C.c_int64, [C.c_void_p]),
    "rt_buf_alloc": (C.c_int, [C.c_void_p, C.c_size_t, C.POINTER(C.c_void_p)]),
    "rt_buf_free": (C.c_int, [C.c_void_p, C.c_void_p]),
    "rt_buf_upload": (C.c_int, [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p, C.c_size_t]),
    "rt_buf_download": (C.c_int, [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p, C.c_size_t]),
    "rt_attn": (C.c_int, [C.c_void_p, C.POINTER(AttnArgs)]),
    "rt_attn_route": (C.c_int, [C.c_void_p, C.POINTER(AttnArgs), C.POINTER(C.c_char_p)]),
    "rt_attn_decode": (C.c_int, [C.c_void_p, C.POINTER(DecodeArgs)]),
    "rt_attn_decode_noalloc": (C.c_int, [C.POINTER(DecodeArgs), C.c_void_p]),
    "rt_attn_decode_noalloc_status": (C.c_int, [C.c_void_p]),
    "rt_xmem_create": (C.c_int, [C.c_int, C.c_int32, C.c_int32, C.c_int32, C.c_int32, C.c_int32,
                                 C.POINTER(C.c_void_p)]),
    "rt_xmem_export": (C.c_int, [C.c_void_p, C.c_void_p]),
    "rt_xmem_import": (C.c_int, [C.c_void_p, C.c_int32, C.c_void_p]),
    "rt_xmem_attach": (C.c_int, [C.c_void_p, C.c_int32, C.c_void_p]),
    "rt_xmem_exchange": (C.c_int, [C.c_void_p, C.POINTER(Exchange)]),
    "rt_xmem_destroy": (C.c_int, [C.c_void_p]),
    "rt_attn_merge_partials": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_int64, C.c_int32,
                                         C.c_void_p, C.c_int32]),
    "rt_rope": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64,
                          C.c_int64, C.c_int32, C.c_int64, C.c_int64, C.c_int32]),
    "rt_matmul": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                            C.c_int64, C.c_int64, C.c_int64, C.c_int64, C.c_int64, C.c_int32,
                            C.c_int32]),
    "rt_argmax_dot": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64,
                                C.c_int64, C.c_int32]),
    "rt_local_attention": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                     C.c_int64, C.c_int32, C.c_int32, C.c_int32, C.c_float,
                                     C.c_float, C.c_int32]),
    "rt_softmax": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_int64,
                             C.c_int32, C.c_int32, C.c_int32]),
    "rt_slice": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int64,
                           C.c_int64, C.c_int64, C.c_int64, C.c_int32]),
    "rt_windows": (C.c_int, [C.c_void_p, C.POINTER(Window), C.c_int32, C.c_int32]),
    "rt_kv_append": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_int64,
                               C.c_int64, C.c_int64, C.c_int32]),
    "rt_rotary": (C.c_int, [C.c_void_p, C.POINTER(RotaryArgs)]),
    "rt_attn_tree": (C.c_int, [C.c_void_p, C.POINTER(TreeArgs)]),
    "rt_attn_tree_route": (C.c_int, [C.c_void_p, C.POINTER(TreeArgs), C.POINTER(C.c_char_p)]),
    "rt_verify_drafts": (C.c_int, [C.c_void_p, C.POINTER(VerifyArgs)]),
    "rt_commit_rows": (C.c_int, [C.c_void_p, C.POINTER(CommitArgs)]),
    "rt_commit_rows_counted": (C.c_int, [C.c_void_p, C.POINTER(CommitCountedArgs)]),
}

# What csrc/host.cpp calls, in the order of its table.
HOST_CALLS = ("rt_matmul", "rt_rope", "rt_slice", "rt_attn", "rt_attn_route", "rt_attn_decode",
              "rt_argmax_dot", "rt_kv_append", "rt_softmax", "rt_windows")

try:
    from . import _host as host   # constructors and eval loop in native code
except ImportError:               # not built: the Python they stand for runs
    host = None

_lib = None


def load():
    """The loaded library, or NOT_INITIALIZED if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RunntimeError(
                "NOT_INITIALIZED",
                f"{LIB_PATH} is missing: build it with `python -m runntime_b200.build` "
                "(there is no CPU fallback)")
        lib = C.CDLL(LIB_PATH)
        for name, (res, args) in SYMBOLS.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        bind_host(lib)
        _lib = lib
    return _lib


def address(x) -> Optional[int]:
    """A device address: None, an int, or a tensor's."""
    if x is None or isinstance(x, int):
        return x
    return int(x.data_ptr())


def call(lib, name: str, ctx, cls, *values) -> None:
    """``name(ctx, structure)`` with the fields of ``cls`` in order; addresses as ``address`` takes them.  In
    native code where it is built: a structure of thirty fields takes ctypes 4 us."""
    fn = getattr(lib, name)
    if host is not None:
        at = _addresses.get((lib, name))
        if at is None:
            at = _addresses[lib, name] = C.cast(fn, C.c_void_p).value
        status = host.call(at, ctx.value, cls.layout, *values)
    else:
        kept, made = [], cls()
        for (field, _), kind, v in zip(cls._fields_, cls.layout, values, strict=True):
            if kind == "A":
                kept.append((C.c_void_p * len(v))(*map(address, v)))
                v = C.cast(kept[-1], C.POINTER(C.c_void_p))
            setattr(made, field, address(v) if kind == "P" else v)
        status = fn(ctx, C.byref(made))
    if status:
        check(status, ctx)


_addresses: dict = {}


def bind_host(lib) -> None:
    """The library that csrc/host.cpp calls; executors of another one run in Python."""
    if host is not None:
        host.bind_library(lib, tuple(C.cast(getattr(lib, n), C.c_void_p).value for n in HOST_CALLS))


def check(status: int, ctx=None):
    """Raises RunntimeError for a non-zero rt_status."""
    if status != 0:
        msg = load().rt_last_error(ctx)
        raise RunntimeError(code_of_status(status), (msg or b"").decode("utf-8", "replace"))
