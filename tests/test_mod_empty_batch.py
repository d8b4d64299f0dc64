"""ln_mod_backward of no images, with modulation rows of either shape (CPU: nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from selas_b200 import build, ops


@pytest.mark.parametrize("shape", [(0, 64), (0, 1, 64)])
def test_no_images(monkeypatch, shape):
    build.build()
    monkeypatch.setattr(ops, "_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_launch", lambda *a: pytest.fail("launched"))
    x = torch.zeros(0, 5, 64)
    dx, dshift, dscale = ops.ln_mod_backward(x, x, torch.zeros(shape, dtype=torch.bfloat16))
    assert dx.shape == x.shape and dshift.shape == dscale.shape == (0, 64)
