"""Host arrays on machines that lock no memory that already exists: pin() leaves them pageable, unpin() takes them back."""
import mmap
import os

import numpy as np
import pytest

from poreplex_amd import native


class Library:
    """The two calls of the C ABI, answering with `code`."""

    def __init__(self, code):
        self.code, self.released = code, []

    def pxg_host_register(self, handle, ptr, nbytes):
        return self.code

    def pxg_host_unregister(self, handle, ptr):
        self.released.append(ptr.value)
        return 0

    def pxg_last_error(self, handle):
        return b'the reason'

    def pxg_destroy(self, handle):
        return 0


def context(code):
    ctx = object.__new__(native.NativeContext)
    ctx.lib, ctx.handle = Library(code), 1
    return ctx


def pages():
    return np.frombuffer(mmap.mmap(-1, 1 << 16), dtype=np.int16)


def test_an_array_that_is_not_locked_stays_usable():
    ctx, array = context(native.PXG_E_UNSUPPORTED), pages()
    assert ctx.pin(array) is array
    ctx.unpin(array)
    assert ctx.lib.released == []
    ctx.lib.code = 0                                   # the same address, locked this time
    ctx.pin(array)
    ctx.unpin(array)
    assert ctx.lib.released == [array.ctypes.data]


def test_a_lock_is_released_whatever_was_refused_at_its_address():
    ctx, array = context(native.PXG_E_UNSUPPORTED), pages()
    ctx.pin(array)                                     # refused, and gone without unpin()
    ctx.lib.code = 0
    ctx.pin(array)                                     # what is mapped there now is locked
    ctx.unpin(array)
    assert ctx.lib.released == [array.ctypes.data] and not ctx._pinned and not ctx._unlocked


def test_arrays_that_stay_pageable_are_said_to(monkeypatch):
    monkeypatch.setattr(native, '_warned_of_pageable', False, raising=False)
    with pytest.warns(RuntimeWarning, match='pageable') as seen:
        for _ in range(3):
            ctx, array = context(native.PXG_E_UNSUPPORTED), pages()
            ctx.pin(array)
            ctx.unpin(array)
    assert len(seen) == 1                              # once in a process


def test_pageable_memory_has_no_way_to_the_runtime():
    """The runtime's own lock of a pageable range can end the process in a GPU memory fault: no switch leads there, and nothing in the
    tree builds device code for, or repeats runs until, such a fault."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    csrc = os.path.join(root, 'poreplex_amd', 'csrc')
    with open(os.path.join(csrc, 'pxg_api.hip')) as f:
        source = f.read()
    begin = source.index('int pxg_h2d_big(')
    assert 'getenv("PXG_H2D' not in source and 'LOCKS")' not in source[begin:source.index('\n}\n', begin)]
    with open(os.path.join(csrc, 'Makefile')) as f:
        assert 'xnack' not in f.read()
    for folder, _, names in os.walk(os.path.join(root, 'tools')):
        for name in names:
            assert not name.endswith('hunt.sh')
            if name.endswith(('.sh', '.py')):
                with open(os.path.join(folder, name)) as f:
                    assert 'HSA_XNACK' not in f.read(), name


def test_other_errors_are_raised():
    with pytest.raises(native.PxgError, match='the reason'):
        context(-3).pin(pages())


@pytest.mark.gpu
def test_a_refused_lock_leaves_no_error_behind():
    from poreplex_amd.config import default_config
    ctx = native.NativeContext(default_config())
    array = pages()
    ctx.pin(array)
    ctx.unpin(array)
    other = native.NativeContext(default_config())     # a stale error would end this call
    other.close()
    ctx.close()


@pytest.mark.gpu
def test_a_wrong_range_is_an_error_of_its_own():
    from poreplex_amd.config import default_config
    ctx = native.NativeContext(default_config())
    array = pages()
    register = ctx.lib.pxg_host_register
    for at, size in ((array.ctypes.data, 1 << 40), (4096, 4096), (array.ctypes.data, (1 << 64) - 1)):    # not mapped (all of it)
        assert register(ctx.handle, at, size) == -1
    rc = register(ctx.handle, array.ctypes.data, array.nbytes)
    assert rc in (0, native.PXG_E_UNSUPPORTED)
    if rc == 0:
        assert ctx.lib.pxg_host_unregister(ctx.handle, array.ctypes.data) == 0
    ctx.close()
