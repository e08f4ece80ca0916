"""HipBackend's wrappers of storage handles, with stand-ins of the library."""
from __future__ import annotations

import types
import weakref

from orcaml_amd import _lib
from orcaml_amd.backend import HipStorage


def test_a_wrapper_is_out_of_sight_before_its_handle_is_released():
    """The release lets other threads run: one that is given the same handle for a new storage must not find
    the dying wrapper."""
    seen = []

    def release(h):
        r = be._live.get(h)
        seen.append((h, None if r is None else r()))
        return _lib.OK

    be = types.SimpleNamespace(_live={}, ctx=types.SimpleNamespace(handle=1), _release_fn=release)
    w = HipStorage(be, 5)
    be._live[5] = weakref.ref(w)
    del w
    assert seen == [(5, None)] and 5 not in be._live


def test_a_second_wrapper_of_the_handle_stays():
    be = types.SimpleNamespace(_live={}, ctx=types.SimpleNamespace(handle=1), _release_fn=lambda h: _lib.OK)
    w, other = HipStorage(be, 5), HipStorage(be, 5)
    be._live[5] = weakref.ref(other)
    del w
    assert be._live[5]() is other
