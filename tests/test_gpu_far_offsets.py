"""Token-wise operators on tensors whose rows lie more than 2^31 elements apart, and on vectors that start off their
alignment: the bits of the same call on compact tensors, or the formula in 64 bits."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from .conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a B200")]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: 0, F16: 1, BF16: 2}
DEV = "cuda"
FAR = (1 << 30) + 8  # a stride that keeps 16-byte rows; three steps of it pass 2^31 elements
WIDE = (1 << 24) + 8  # the same for hundreds of rows


@pytest.fixture(scope="module", autouse=True)
def _lib_ready():
    from selas_b200 import _lib

    _lib.lib()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0, "a kernel reported a device-side error"


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()  # a test holds up to 40 GB


def ops():
    from selas_b200 import ops as o

    return o


def call(entry, args):
    from selas_b200 import _lib

    _lib.check(getattr(_lib.lib(), entry)(ctypes.addressof(args), torch.cuda.current_stream().cuda_stream), entry)


def randn(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def far(t, dim, stride):
    """A copy of the compact tensor t in a buffer of its own, with the given stride along dim."""
    strides = [stride if i == dim else s for i, s in enumerate(t.stride())]
    size = 1 + sum((n - 1) * s for n, s in zip(t.shape, strides))
    return torch.empty(size, dtype=t.dtype, device=DEV).as_strided(t.shape, strides).copy_(t)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("dim", [96, 1000, 16388])
@pytest.mark.parametrize("along", [0, 1])
def test_norm_rows_far_apart(xt, dim, along):
    from selas_b200 import _lib

    g = torch.Generator(device=DEV).manual_seed(60)
    shape = (5, 2, dim) if along == 0 else (1, 5, dim)
    x, dy, w, b = randn(g, *shape, dtype=xt), randn(g, *shape, dtype=BF16), randn(g, dim, mean=1.0), randn(g, dim)
    want, grads = ops().layer_norm(x, w, b), ops().layer_norm_backward(dy, x, w, add=x)
    fx = far(x, along, FAR)
    assert torch.equal(ops().layer_norm(fx, w, b), want)
    assert same(ops().layer_norm_backward(far(dy, along, FAR), fx, w, add=fx), grads)
    out = far(torch.zeros_like(x), along, FAR)
    a = _lib.FbLayerNormArgs()
    a.x, a.out, a.weight, a.bias = fx.data_ptr(), out.data_ptr(), w.data_ptr(), b.data_ptr()
    a.x_outer_stride, a.x_inner_stride = fx.stride()[:2]
    a.out_outer_stride, a.out_inner_stride = out.stride()[:2]
    (a.outer, a.inner, a.dim), a.eps = x.shape, 1e-5
    a.x_dtype, a.y_dtype, a.w_dtype = CODE[xt], CODE[xt], CODE[F32]
    call("fb_layer_norm", a)
    assert torch.equal(out, want)


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("along", [0, 1, 2])
@pytest.mark.parametrize("hd,axes", [(64, (16, 24, 24)), (10, (4, 2, 4))])
def test_rope_rows_far_apart(pairs, along, hd, axes):
    from selas_b200 import _lib

    g = torch.Generator(device=DEV).manual_seed(61)
    shape = [2, 2, 2, hd]
    shape[along] = 5
    x = randn(g, *shape, dtype=BF16)
    ids = torch.randint(0, 90, (shape[2], 3), generator=g, device=DEV)
    want = ops().rope_axes(x, ids, axes, pairs=pairs)
    fx, out = far(x, along, FAR), far(torch.zeros_like(x), along, FAR)
    assert torch.equal(ops().rope_axes(fx, ids, axes, pairs=pairs), want)
    a = _lib.FbRopeArgs()
    a.tensor[0] = _lib.FbRopeTensor(fx.data_ptr(), out.data_ptr(), *fx.stride()[:3], *out.stride()[:3], shape[1])
    a.ids, a.ids_stride_l, a.ids_stride_a, a.ids_type = ids.data_ptr(), 3, 1, _lib.FB_IDS_I64
    a.axes_dim[:3], a.theta[:3] = axes, (10000.0,) * 3
    a.count, a.dtype, a.batch, a.seq, a.head_dim, a.axes = 1, CODE[BF16], shape[0], shape[2], hd, 3
    a.pairs = ("interleaved", "halves").index(pairs)
    call("fb_rope_axes", a)
    assert torch.equal(out, want)


def test_rope_ids_far_apart():
    g = torch.Generator(device=DEV).manual_seed(62)
    x = randn(g, 1, 2, 5, 64, dtype=BF16)
    ids = torch.randint(0, 90, (5, 3), generator=g, device=DEV, dtype=torch.int32)
    assert torch.equal(ops().rope_axes(x, far(ids, 0, FAR), (16, 24, 24)), ops().rope_axes(x, ids, (16, 24, 24)))


@pytest.mark.parametrize("m,n,k,stride", [(5, 300, 256, FAR), (300, 20000, 64, WIDE)])
def test_linear_rows_far_apart(m, n, k, stride):
    """Inputs, residual and output; few rows, and the pair kernel."""
    from selas_b200 import _lib

    g = torch.Generator(device=DEV).manual_seed(63)
    x, w, b, r = randn(g, m, k, dtype=BF16), randn(g, n, k, dtype=BF16, std=1 / math.sqrt(k)), randn(g, n, dtype=BF16), randn(g, m, n, dtype=BF16)
    want = ops().linear_act(x, w, b, "gelu", r)
    fx, fr = far(x, 0, stride), far(r, 0, stride)
    assert torch.equal(ops().linear_act(fx, w, b, "gelu", fr), want)
    out = far(torch.zeros_like(r), 0, stride)
    a = _lib.FbLinearActArgs()
    a.x, a.ldx, a.w, a.ldw, a.bias = fx.data_ptr(), stride, w.data_ptr(), k, b.data_ptr()
    a.residual, a.ld_residual, a.out, a.ld_out = fr.data_ptr(), stride, out.data_ptr(), stride
    a.m, a.n, a.k = m, n, k
    a.dtype, a.residual_dtype, a.out_dtype, a.act = CODE[BF16], CODE[BF16], CODE[BF16], _lib.FB_ACT_GELU
    call("fb_linear_act", a)
    assert torch.equal(out, want)
    # off 16 bytes: x is copied first, outputs go one by one; the last bits may differ from those of whole vectors
    z = torch.nn.functional.gelu(x.double() @ w.double().t() + b.double()) + r.double()
    s = x.double().abs() @ w.double().abs().t() + b.double().abs()
    off = ops().linear_act(far(x, 0, stride + 1), w, b, "gelu", far(r, 0, stride + 3)).double()
    assert ((off - z).abs() <= 1.13 * (k / 16 + 8) * 2.0 ** -22 * s + 2.0 ** -20 * (s + r.double().abs()) + z.abs() * 2.0 ** -8 * (1 + 2.0 ** -8)).all()


@pytest.mark.parametrize("m,n,k", [(3, 300, 64), (200, 333, 520), (600, 1024, 8192), (300, 20000, 64)])
@pytest.mark.parametrize("start", [1, 2, 4])
def test_linear_vectors_off_alignment(m, n, k, start):
    """A bias and a residual that start 2, 4 or 8 bytes past a 16-byte boundary."""
    g = torch.Generator(device=DEV).manual_seed(64)
    x, w = randn(g, m, k, dtype=BF16), randn(g, n, k, dtype=BF16, std=1 / math.sqrt(k))
    b, r = randn(g, n + start, dtype=BF16)[start:], randn(g, m * n + start, dtype=BF16)[start:].view(m, n)
    z = torch.nn.functional.silu(x.double() @ w.double().t() + b.double()) + r.double()
    s = x.double().abs() @ w.double().abs().t() + b.double().abs()
    for residual in (r, None):
        got = ops().linear_act(x, w, b, "silu", residual).double()
        ref = z if residual is not None else z - r.double()
        assert ((got - ref).abs() <= 1.13 * (k / 16 + 8) * 2.0 ** -22 * s + 2.0 ** -20 * (s + r.double().abs()) + ref.abs() * 2.0 ** -8 * (1 + 2.0 ** -8)).all()


@pytest.mark.parametrize("dim", [24, 64, 128, 1024, 3072, 12288])
@pytest.mark.parametrize("wt", [BF16, F32])
def test_norm_weights_off_alignment(dim, wt):
    """Weight, bias and modulation rows that start one element past their vector's boundary, whole rows besides: against the
    same values at an aligned place. Both orders of the sums are off by at most 32 u of a mean magnitude, here some 2e-6 of
    values of size ten; the sums of 40 rows by (64 + 24) u of their magnitudes."""
    g = torch.Generator(device=DEV).manual_seed(65)
    x, dy = randn(g, 4, 10, dim), randn(g, 4, 10, dim)
    w, b = randn(g, dim + 1, std=0.3, mean=1.0, dtype=wt)[1:], randn(g, dim + 1, dtype=wt)[1:]
    near = lambda p, q: all(((s - t).abs() <= 4e-5).all() and s.isfinite().all() for s, t in zip(p, q))  # noqa: E731
    assert near((ops().layer_norm(x, w, b),), (ops().layer_norm(x, w.clone(), b.clone()),))
    assert near(ops().layer_norm_backward(dy, x, w), ops().layer_norm_backward(dy, x, w.clone()))
    scale = randn(g, 4, 6 * dim + 1, std=0.3, dtype=BF16)[:, 1:dim + 1]
    assert near(ops().ln_mod_backward(dy, x, scale), ops().ln_mod_backward(dy, x, scale.clone()))
