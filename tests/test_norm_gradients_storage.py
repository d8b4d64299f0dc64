"""What the gradients of the norms hold on to (CPU: the wrappers allocate before the launch, which is left out here)."""

from __future__ import annotations

import pytest
import torch

from selas_b200 import _lib, ops

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def recorded(monkeypatch):
    from selas_b200 import build

    build.build()
    packed = []
    monkeypatch.setattr(ops, "_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_launch", lambda index, entry, flops, nbytes, args: packed.append(args))
    return packed


@pytest.mark.parametrize("rows,d", [(1, 64), (5, 64), (600, 768), (4, 20000)])
def test_gradients_keep_only_themselves(recorded, rows, d):
    """dweight and dbias, and dscale and dshift, each own exactly their values: no workspace lives on with them, and
    saving or keeping one does not keep the other."""
    x = torch.zeros(2, rows, d)
    for grads in (ops.layer_norm_backward(x, x, torch.ones(d))[1:], ops.ln_mod_backward(x, x, torch.ones(2, d, dtype=BF16))[1:]):
        for t in grads:
            assert t.dtype == torch.float32 and t.is_contiguous()
            assert t.untyped_storage().nbytes() == 4 * t.numel()
        assert grads[0].untyped_storage().data_ptr() != grads[1].untyped_storage().data_ptr()
    assert len(recorded) == 2


def test_the_kernel_gets_the_gradients_and_its_workspace(recorded):
    x = torch.zeros(2, 600, 768)
    for call, groups in ((lambda: ops.layer_norm_backward(x, x)[1:], 1), (lambda: ops.ln_mod_backward(x, x, torch.ones(2, 768, dtype=BF16))[:0:-1], 2)):
        dw, db = call()
        a = _lib.FbLayerNormArgs.from_buffer_copy(recorded.pop())
        assert (a.dweight, a.dbias) == (dw.data_ptr(), db.data_ptr())
        need = _lib.load().fb_layer_norm_work_floats(2, 600, 768, groups > 1)
        assert a.work_floats == need > 0 and a.work not in (None, a.dweight, a.dbias)
