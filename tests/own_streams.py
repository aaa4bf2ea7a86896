"""HIP streams of a test's own, default priority.  PyTorch hands out its pool's 32 in turn, so each taken from there moves which
of them a later test gets, and with it whether calls that keep something by stream have seen it: tests/test_zz_no_alloc.py captures on two
that no earlier call may have used.  A test that only needs another stream takes one from here."""
import ctypes
import functools
import os

import torch


@functools.lru_cache(None)
def stream(n=0):
    """The n-th of them, made once and kept until the process ends."""
    hip = ctypes.CDLL(os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so"))
    handle = ctypes.c_void_p()
    error = hip.hipStreamCreateWithFlags(ctypes.byref(handle), ctypes.c_uint(1))  # (does not wait for the null stream)
    assert error == 0, error
    return torch.cuda.ExternalStream(handle.value)
