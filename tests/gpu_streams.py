"""A stream that no call has used yet: torch's own come from a pool and are handed out again, to other tests, too."""
import ctypes

import torch

from izwi_amd import capi


def fresh_stream() -> torch.cuda.ExternalStream:
    """Of default priority, alive until the process ends.  (By the HIP runtime that the library is linked to.)"""
    handle = ctypes.c_void_p()
    rc = capi.lib().hipStreamCreate(ctypes.byref(handle))
    assert rc == 0 and handle.value, rc
    return torch.cuda.ExternalStream(handle.value)
