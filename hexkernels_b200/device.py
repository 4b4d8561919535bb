"""Device-pointer launchers over libhexcuda (asynchronous, inputs resident in
HBM).  Arguments may be torch CUDA tensors (their data_ptr() is passed) or raw
integer device addresses; scalars pass through.  ``bind_stream`` makes the
launches go to torch's current stream so torch.cuda.Event timing brackets them.
"""
from __future__ import annotations

import ctypes as C

from ._lib import check, load


_PLAIN = frozenset((int, float, type(None)))
_entries: dict[str, C._CFuncPtr] = {}


def _arg(a):
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    return a


def launch(name: str, dev: int, *args) -> None:
    """Call ``hexcuda_<name>(dev, *args)``; raises on a non-zero status."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(load(), "hexcuda_" + name)
    # (a small launch is bound by this call: numbers are told apart by type
    # alone, and the rest is taken for a tensor first)
    try:
        values = [a if type(a) in _PLAIN else a.data_ptr() for a in args]
    except AttributeError:
        values = [_arg(a) for a in args]
    rc = fn(dev, *values)
    if rc:
        check(rc)


def bind_stream(dev: int, stream=None) -> None:
    """Route device `dev`'s launches to a torch stream (default: current)."""
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    check(load().hexcuda_set_stream(dev, s.cuda_stream))


def paged_attn_workspace(dev: int) -> int:
    """Bytes of device memory that a ``paged_attn`` call takes as workspace."""
    n = C.c_size_t()
    check(load().hexcuda_paged_attn_workspace(dev, C.byref(n)))
    return n.value


def sync(dev: int = -1) -> None:
    check(load().hexcuda_sync(dev))


def launch_count() -> int:
    return int(load().hexcuda_launch_count())
