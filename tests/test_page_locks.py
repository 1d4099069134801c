"""Host arrays on machines that lock no memory that already exists: pin() leaves them pageable, unpin() takes them back."""
import mmap

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
