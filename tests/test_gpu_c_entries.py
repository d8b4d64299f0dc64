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


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("hd,axes", [(64, (16, 24, 24)), (128, (16, 56, 56)), (10, (4, 6)), (80, (10, 30, 40))])
def test_rope_in_place(pairs, dt, hd, axes):
    """q and k turned where they are, inside a fused projection's rows: the bits of the turn beside them, and what else
    the rows hold stays."""
    from selas_b200 import _lib, ops

    g = torch.Generator(device=DEV).manual_seed(51)
    for b, l, h, kv, pad in ((1, 1, 24, 24, 0), (2, 45, 6, 2, 0), (1, 3001, 5, 1, 0), (2, 37, 3, 3, 3)):
        width = (h + 2 * kv) * hd + pad
        rows = randn(g, b, l, width, dtype=dt)
        heads = rows[..., :(h + 2 * kv) * hd].unflatten(-1, (h + 2 * kv, hd))
        q, k = heads[:, :, :h].transpose(1, 2), heads[:, :, h:h + kv].transpose(1, 2)
        ids = torch.randint(0, 90, (l, len(axes)), generator=g, device=DEV)
        wq, wk = ops.rope_axes_qk(q, k, ids, axes, pairs=pairs)
        rest = rows[..., (h + kv) * hd:].clone()
        a = _lib.FbRopeArgs()
        for i, (t, n) in enumerate(((q, h), (k, kv))):
            st = t.stride()[:3]
            a.tensor[i] = _lib.FbRopeTensor(t.data_ptr(), t.data_ptr(), *st, *st, n)
        a.ids, a.ids_stride_l, a.ids_stride_a, a.ids_type = ids.data_ptr(), len(axes), 1, _lib.FB_IDS_I64
        a.axes_dim[:len(axes)], a.theta[:len(axes)] = axes, (10000.0,) * len(axes)
        a.count, a.dtype, a.batch, a.seq, a.head_dim, a.axes = 2, CODE[dt], b, l, hd, len(axes)
        a.pairs = _lib.FB_ROPE_INTERLEAVED if pairs == "interleaved" else _lib.FB_ROPE_HALVES
        call("fb_rope_axes", a)
        assert torch.equal(q, wq) and torch.equal(k, wk) and torch.equal(rows[..., (h + kv) * hd:], rest)


@pytest.mark.parametrize("m,n,k", [(1, 300, 256), (28, 3072, 3072), (77, 1001, 512), (333, 1111, 1000), (2000, 640, 128), (2601, 4004, 424), (2601, 4003, 424),
                                   (500, 1020, 8456), (500, 1019, 8456)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_residual_in_the_place_of_out(m, n, k, dt):
    """The output written over the residual, with a row stride of its own, has the bits of an output of that stride beside it
    (with another stride the bias may be added in another order)."""
    from selas_b200 import _lib

    g = torch.Generator(device=DEV).manual_seed(52)
    x, w, b = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, std=k ** -0.5), randn(g, n, dtype=dt)
    for out_type in (dt, F32):
        for ld in (n, n + 4, n + 3):
            room = randn(g, m, ld, dtype=out_type)
            res, after, beside = room[:, :n], room[:, n:].clone(), torch.zeros_like(room)
            for out in (beside, room):
                a = _lib.FbLinearActArgs()
                a.x, a.ldx, a.w, a.ldw, a.bias = x.data_ptr(), k, w.data_ptr(), k, b.data_ptr()
                a.residual, a.ld_residual, a.out, a.ld_out = res.data_ptr(), ld, out.data_ptr(), ld
                a.m, a.n, a.k = m, n, k
                a.dtype, a.residual_dtype, a.out_dtype, a.act = CODE[dt], CODE[out_type], CODE[out_type], _lib.FB_ACT_GELU
                call("fb_linear_act", a)
            assert torch.equal(res, beside[:, :n]) and torch.equal(room[:, n:], after) and not beside[:, n:].any()
            y = torch.nn.functional.gelu(x.double() @ w.double().t() + b.double())
            assert beside[:, :n].isfinite().all() and (beside[:, :n] - y).norm() > 0.5 * y.norm()  # the residual is in it


@pytest.mark.parametrize("dim", [8, 24, 64, 77, 128, 1000, 3072, 16388])
@pytest.mark.parametrize("xt,wt", [(F32, BF16), (BF16, F32), (F16, F16)])
def test_norm_with_a_weight_row_per_outer_index(dim, xt, wt):
    """fb_layer_norm with weight and bias rows of their own per outer index (strided), as scale (1 + weight) and as weight,
    against the formula in 64 bits: groups of threads that share a warp stand at different outer indices. Bounds as for
    one weight: a centred value is off by 32 u mean|x| + 2 u |x|, rstd by 24 u relative, and product and sum add three
    roundings (u = 2^-24) and the output's half step."""
    from selas_b200 import _lib

    g = torch.Generator(device=DEV).manual_seed(53)
    u = 2.0 ** -24
    for outer, inner in ((2, 1), (5, 7), (3, 333), (700, 3), (1, 40)):
        if outer * inner * dim > 8_000_000:
            continue
        x = randn(g, outer, inner, dim, dtype=xt, mean=0.3)
        xd = x.double()
        c = xd - xd.mean(-1, keepdim=True)
        rstd = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5)
        h = c * rstd
        dh = u * (32 * rstd * xd.abs().mean(-1, keepdim=True) + 2 * rstd * xd.abs() + 24 * h.abs())
        for pad in (0, 4, 3):
            rows = randn(g, 2, outer, dim + pad, dtype=wt, std=0.3)
            w, b = rows[0, :, :dim], rows[1, :, :dim]
            for plus in (0, 1):
                for has_w, has_b in ((1, 1), (1, 0), (0, 1)):
                    for yt in (xt, BF16):
                        out = torch.empty(outer, inner, dim, dtype=yt, device=DEV)
                        a = _lib.FbLayerNormArgs()
                        a.x, a.out = x.data_ptr(), out.data_ptr()
                        a.weight, a.bias = (w.data_ptr() if has_w else None), (b.data_ptr() if has_b else None)
                        a.x_outer_stride = a.out_outer_stride = inner * dim
                        a.x_inner_stride = a.out_inner_stride = dim
                        a.w_outer_stride, a.weight_plus_one = dim + pad, plus
                        a.outer, a.inner, a.dim, a.eps = outer, inner, dim, 1e-5
                        a.x_dtype, a.y_dtype, a.w_dtype = CODE[xt], CODE[yt], CODE[wt]
                        call("fb_layer_norm", a)
                        wf = (w.double() + plus)[:, None] if has_w else torch.ones(1, device=DEV).double()
                        bf = b.double()[:, None] if has_b else 0.0 * wf
                        ref = h * wf + bf
                        slack = dh * wf.abs() + 3 * u * ((h * wf).abs() + bf.abs())
                        half = ref.abs() * (torch.finfo(yt).eps / 2) + (2.0 ** -25 if yt == F16 else 0.0)
                        worst = ((out.double() - ref).abs() / (slack * (1 + torch.finfo(yt).eps) + half + 1e-37)).max().item()
                        assert worst <= 1.0, (outer, inner, pad, plus, has_w, has_b, yt, worst)
