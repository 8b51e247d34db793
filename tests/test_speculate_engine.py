"""KvCacheEngine's speculative step without a GPU: the structures of its calls, and what it refuses before them."""
import ctypes as C

import runntime_b200._lib as L


def test_counted_commit_is_a_commit_and_an_address():
    assert L.CommitCountedArgs.layout == L.CommitArgs.layout + "P"
    assert L.CommitCountedArgs.committed.offset == C.sizeof(L.CommitArgs)
    for name, _ in L.CommitArgs._fields_:
        assert getattr(L.CommitCountedArgs, name).offset == getattr(L.CommitArgs, name).offset
