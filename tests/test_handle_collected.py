"""Handles that the garbage collector finds, on a library that only counts (no GPU)."""
import os
import subprocess
import sys

import pytest

from aidotnet.tensors_b200 import native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Counting:
    def __init__(self):
        self.destroyed = []

    def aidn_sdpa_destroy(self, h):
        self.destroyed.append(h)

    def aidn_sdpa_poll(self, h, stream):
        return N.OK

    def aidn_sdpa_workspace_bytes(self, h, *sizes):
        return 0

    aidn_sdpa_kv8_workspace_bytes = aidn_sdpa_workspace_bytes


def handle(lib, number):
    h = N.Handle.__new__(N.Handle)
    h._lib, h._h, h._kv8_asked = lib, number, None
    return h


@pytest.mark.parametrize("call", [lambda h: h.workspace_bytes(1, 1, 1), lambda h: h.kv8_workspace_bytes(1, 1, 1), lambda h: h.poll(0)])
def test_collected_in_a_capture_is_destroyed_by_the_next_call(monkeypatch, call):
    lib, busy = Counting(), [True]
    monkeypatch.setattr(N, "_capturing", lambda: busy[0])
    kept = handle(lib, 1)
    handle(lib, 2).__del__()
    call(kept)
    assert lib.destroyed == []
    busy[0] = False
    call(kept)
    assert lib.destroyed == [2] and not N._left
    kept.close()
    assert lib.destroyed == [2, 1]


def test_destroyed_once_and_not_at_all_after_close(monkeypatch):
    lib, busy = Counting(), [True]
    monkeypatch.setattr(N, "_capturing", lambda: busy[0])
    closed, twice = handle(lib, 3), handle(lib, 4)
    closed.close()
    closed.__del__()
    twice.__del__()
    twice.__del__()
    busy[0] = False
    N._destroy_left()
    assert lib.destroyed == [3, 4]


def test_destroyed_where_torch_cannot_be_asked(monkeypatch):
    def gone():
        raise AttributeError("torch has been taken down")

    lib = Counting()
    monkeypatch.setattr(N, "_capturing", gone)
    handle(lib, 5).__del__()
    assert lib.destroyed == [5]


def test_destroyed_at_the_interpreter_s_end():
    code = ("from aidotnet.tensors_b200 import native as N\n"
            "class Lib:\n"
            "    def aidn_sdpa_destroy(self, h): print('destroyed', h, flush=True)\n"
            "N._left.append((Lib(), 6))\n")
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, check=True).stdout
    assert out.split() == ["destroyed", "6"]
