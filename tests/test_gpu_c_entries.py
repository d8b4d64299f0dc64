"""Forms of the token-wise operators that the C interface has beside those of the wrappers: outputs in the place of an input,
and the forward norm with a weight row per outer index."""

from __future__ import annotations

import ctypes

import pytest
import torch

from .conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a B200")]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: 0, F16: 1, BF16: 2}
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib_ready():
    from selas_b200 import _lib

    _lib.lib()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0, "a kernel reported a device-side error"


def randn(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def call(entry, args):
    from selas_b200 import _lib

    _lib.check(getattr(_lib.lib(), entry)(ctypes.addressof(args), torch.cuda.current_stream().cuda_stream), entry)


@pytest.mark.parametrize("xt", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [24, 64, 77, 1000, 1001, 2304, 6144, 12288, 16384, 20004])
def test_dx_in_the_place_of_add(dim, xt):
    """dx written over add, also where rows are strided, has the bits of dx beside it."""
    from selas_b200 import _lib, ops

    g = torch.Generator(device=DEV).manual_seed(50)
    for outer, inner, ld in ((1, 3, dim), (2, 300, dim), (3, 70, dim + 5), (2, 40, dim + 4)):
        x, dy, w = randn(g, outer, inner, dim, dtype=xt), randn(g, outer, inner, dim, dtype=BF16), randn(g, dim, mean=1.0)
        room = randn(g, outer, inner, ld, dtype=xt)
        add = room[..., :dim]
        want, after = ops.layer_norm_backward(dy, x, w, add=add, sums=False)[0], room[..., dim:].clone()
        a = _lib.FbLayerNormArgs()
        a.x, a.dy, a.add, a.out, a.weight = x.data_ptr(), dy.data_ptr(), add.data_ptr(), add.data_ptr(), w.data_ptr()
        a.x_outer_stride, a.x_inner_stride = a.dy_outer_stride, a.dy_inner_stride = inner * dim, dim
        a.add_outer_stride, a.add_inner_stride = a.out_outer_stride, a.out_inner_stride = inner * ld, ld
        a.outer, a.inner, a.dim, a.eps = outer, inner, dim, 1e-5
        a.x_dtype, a.y_dtype, a.w_dtype = CODE[xt], CODE[BF16], CODE[F32]
        call("fb_layer_norm_backward", a)
        assert torch.equal(add, want) and torch.equal(room[..., dim:], after)
