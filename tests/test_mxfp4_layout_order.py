"""Weights in the microscaled four-bit format are published in the kernels' layout once they lie in it (host logic, on the CPU: the launches are recorded)."""
from types import SimpleNamespace

import pytest
import torch

from hibana_amd import _lib
from hibana_amd.kernels import mxfp4, mxfp4_moe
from hibana_amd.weights.mxfp4 import Mxfp4Linear


@pytest.fixture
def steps(monkeypatch):
    """What is enqueued and waited for, in order; each with whether the weights were published by then."""
    done, seen = [], SimpleNamespace(published=lambda: None)
    real = _lib.lib()
    fake = SimpleNamespace(hb_mxfp4_tiled_bytes=real.hb_mxfp4_tiled_bytes, hb_mxfp4_repack=lambda *a: done.append(("layout", seen.published())) or 0)
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(_lib, "need_one_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "stream", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: SimpleNamespace(synchronize=lambda: done.append(("wait", seen.published()))))
    seen.done = done
    return seen


def _held(*shape):
    *lead, n, k = shape
    return torch.zeros(*lead, n, k // 2, dtype=torch.uint8), torch.zeros(*lead, n, k // 32, dtype=torch.uint8)


def test_a_linears_layout_is_waited_for_ahead_of_its_use(steps):
    lin = Mxfp4Linear(*_held(64, 96))
    steps.published = lambda: lin.tiled is not None or lin.codes is None
    lin.tile(release=True)
    assert steps.done == [("layout", False), ("wait", False)]
    assert lin.tiled is not None and lin.codes is None


def test_the_experts_layouts_are_waited_for_ahead_of_their_use(steps):
    ex = mxfp4_moe.Mxfp4Experts(*_held(3, 64, 96), *_held(3, 96, 32))
    steps.published = lambda: (ex.tiled1 is not None) + (ex.tiled2 is not None) + 2 * (ex.fc1_codes is None)
    mxfp4_moe.tile(ex, release=True)
    assert steps.done == [("layout", 0), ("wait", 0), ("layout", 1), ("wait", 1)]
    assert ex.tiled2 is not None and ex.fc2_codes is None


def test_many_matrices_are_waited_for_once(steps):
    mxfp4.tile(mxfp4.Mxfp4(*_held(65536, 1, 32)))
    assert [what for what, _ in steps.done] == ["layout", "layout", "wait"]
