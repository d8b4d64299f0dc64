"""The token-wise operators on a B200 against their formulas in 64 bits: rotary positions with several axes
(ops.rope_axes), layer norm and its gradients (ops.layer_norm, layer_norm_backward, ln_mod_backward) and the Linear with
activation and residual (ops.linear_act).

Every check is elementwise against a bound worked out beforehand. With u = 2^-24 (half a step of fp32) and h the half
step of the output's type (bf16 2^-8, fp16 2^-11, fp32 2^-24, relative; fp16 also 2^-25 absolute below its normal
range), the bounds count:
  rope       the angle's fraction of a turn rounded to fp32 (2^-26 turns = 0.8 * 2^-23 rad), one step of sincospif, and
             two products and a sum: 4 * 2^-23 * (|a| + |b|) for a pair (a, b), plus h |y|;
  norm       sums of D values in chains of at most 32 roundings (16 elements of a thread, five shuffles, the warps):
             the mean is off by 32 u mean|x|, a centred value by that + u |x|, rstd by 20 u relative;
  gradients  the same, carried through the formulas; the column sums add chains of rows per block, blocks and groups;
  linear     the tensor core adds 16 products and the accumulator at a time, off by at most 2^-22 of the sum of
             magnitudes S per step: (K / 16 + 8) 2^-22 S, carried through the activation (slope at most 1.13).
"""

from __future__ import annotations

import math

import pytest
import torch

from .conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a B200")]

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
DEV = "cuda"
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _lib_ready():
    from selas_b200 import _lib

    _lib.lib()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0, "a kernel reported a device-side error"


def ops():
    from selas_b200 import ops as o

    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def half_step(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == F16 else 0.0)


def check(got, ref, slack, name=""):
    """|got - ref| <= slack + the rounding of the output, elementwise (ref in 64 bits)."""
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert torch.isfinite(got).all(), name
    err = (got.double() - ref).abs()
    bound = slack * (1 + torch.finfo(got.dtype).eps) + half_step(ref, got.dtype) + 1e-37
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound, max error {err.max().item():.3g}"


# ------------------------------------------------------------------------------------------ rotary positions


def rope_ref(x, ids, axes, theta, pairs, inverse):
    """(result, |a| + |b| of each element's pair) in 64 bits."""
    thetas = theta if isinstance(theta, tuple) else (theta,) * len(axes)
    w = torch.cat([t ** (-torch.arange(0, d, 2, dtype=F64, device=DEV) / d) for d, t in zip(axes, thetas)])
    at = torch.cat([ids[..., a:a + 1].double().expand(*ids.shape[:-1], d // 2) for a, d in enumerate(axes)], -1)
    ang = at * w * (-1 if inverse else 1)
    ang = ang[:, None] if ids.dim() == 3 else ang
    c, s, x = ang.cos(), ang.sin(), x.double()
    if pairs == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        join = lambda p, q: torch.stack((p, q), -1).flatten(-2)  # noqa: E731
    else:
        a, b = x.chunk(2, -1)
        join = lambda p, q: torch.cat((p, q), -1)  # noqa: E731
    mag = a.abs() + b.abs()
    return join(a * c - b * s, a * s + b * c), join(mag, mag)


def check_rope(got, x, ids, axes, theta=10000.0, pairs="interleaved", inverse=False, name=""):
    ref, mag = rope_ref(x, ids, axes, theta, pairs, inverse)
    assert got.dtype == x.dtype and got.is_contiguous()
    check(got, ref, 4 * 2.0 ** -23 * mag, name)


def grid_ids(g, l, axes, dtype, high):
    ids = torch.randint(-3 if dtype != F32 else 0, high, (l, axes), generator=g, device=DEV)
    return ids.to(dtype)


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("axes", [(2,), (2, 4), (16, 56, 56), (10, 30, 40), (6, 6, 2), (64, 96, 96), (512,), (2, 2, 2, 2, 2, 2, 2, 2)])
def test_rope_types_and_axes(pairs, dt, axes):
    g = gen(1)
    hd = sum(axes)
    for b, h, l, inverse in ((1, 1, 1, False), (2, 3, 37, True), (1, 24, 130, False)):
        x = randn(g, b, h, l, hd, dtype=dt)
        ids = grid_ids(g, l, len(axes), torch.int64, 200)
        got = ops().rope_axes(x, ids, axes, pairs=pairs, inverse=inverse)
        check_rope(got, x, ids, axes, pairs=pairs, inverse=inverse, name=f"{b} {h} {l}")


@pytest.mark.parametrize("ids_dt", [F32, F64, torch.int32, torch.int64])
def test_rope_far_positions_and_bases(ids_dt):
    """Positions of millions (angles reduced in 64 bits), fractions and negatives where the type has them, a base per axis."""
    g = gen(2)
    axes, theta = (16, 24, 24), (10000.0, 500.0, 1e6)
    x = randn(g, 1, 4, 301, 64)
    ids = torch.randint(0, 1 << 23, (301, 3), generator=g, device=DEV).to(ids_dt)
    ids[:4] = torch.tensor([[0, 1, 2], [5_000_000, 0, 7], [1, 8_388_607, 8_000_001], [3, 3, 3]], device=DEV).to(ids_dt)
    if ids_dt != torch.int32:
        ids[5] = torch.tensor([-5, -1_000_000, -2], device=DEV).to(ids_dt)
    if ids_dt.is_floating_point:
        ids[6] = torch.tensor([0.25, 1000.125, -0.5], device=DEV).to(ids_dt)
    for pairs in ("interleaved", "halves"):
        check_rope(ops().rope_axes(x, ids, axes, theta, pairs=pairs), x, ids, axes, theta, pairs)


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_rope_strides(pairs, dt):
    """Slices of a fused projection, token-major rows, rows off 16 bytes, ids per image and with strides of their own;
    q and k of different head counts in one launch; the inputs are left as they were."""
    g = gen(3)
    axes, b, l, h, kv, hd = (16, 24, 24), 2, 45, 6, 2, 64
    rows = randn(g, b, l, h + 2 * kv, hd, dtype=dt)
    q, k = rows[:, :, :h].transpose(1, 2), rows[:, :, h:h + kv].transpose(1, 2)
    before = rows.clone()
    ids = grid_ids(g, l, 3, torch.int64, 90)
    qo, ko = ops().rope_axes_qk(q, k, ids, axes, pairs=pairs)
    check_rope(qo, q, ids, axes, pairs=pairs)
    check_rope(ko, k, ids, axes, pairs=pairs)
    assert torch.equal(rows, before)
    ids3 = torch.stack((ids, ids.flip(0)))
    check_rope(ops().rope_axes(q, ids3, axes, pairs=pairs), q, ids3, axes, pairs=pairs)
    cols = ids.t().contiguous().t()  # column-major
    assert torch.equal(ops().rope_axes(q, cols, axes, pairs=pairs), qo)
    assert torch.equal(ops().rope_axes(q, ids.expand(b, l, 3), axes, pairs=pairs), qo)
    flat = randn(g, b * h * l * hd + 1, dtype=dt)
    off = flat[1:].view(b, h, l, hd)  # rows off 16 bytes
    check_rope(ops().rope_axes(off, ids, axes, pairs=pairs), off, ids, axes, pairs=pairs)
    wide = randn(g, b, h, l, hd + 3, dtype=dt)[..., 2:hd + 2]  # a row stride of its own
    check_rope(ops().rope_axes(wide, ids, axes, pairs=pairs), wide, ids, axes, pairs=pairs)
    same = randn(g, 1, 1, l, hd, dtype=dt).expand(b, h, l, hd)  # one row for every head and image
    check_rope(ops().rope_axes(same, ids, axes, pairs=pairs), same, ids, axes, pairs=pairs)


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("dt,h,kv,axes,l", [(BF16, 24, 24, (16, 56, 56), 4608), (F32, 16, 4, (16, 24, 24), 3001), (F16, 40, 1, (22, 20, 22), 5000),
                                            (BF16, 7, 3, (10, 30, 40), 9001), (F16, 3, 2, (2, 4), 40001)])
def test_rope_many_tokens(pairs, dt, h, kv, axes, l):
    """Enough tokens that a thread takes a run of heads, across the border of q and k, with a run left over."""
    g = gen(7)
    hd = sum(axes)
    q, k = randn(g, 2, h, l, hd, dtype=dt), randn(g, 2, l, kv, hd, dtype=dt).transpose(1, 2)
    ids = grid_ids(g, l, len(axes), F32, 300)
    qo, ko = ops().rope_axes_qk(q, k, ids, axes, pairs=pairs, inverse=True)
    check_rope(qo, q, ids, axes, pairs=pairs, inverse=True)
    check_rope(ko, k, ids, axes, pairs=pairs, inverse=True)


def test_rope_gradient_by_differences():
    """sum(g * rope(x)) along random directions: central differences in fp32 (the map is linear, so a step of one is
    exact up to rounding) against the inverse turn of g."""
    g = gen(4)
    axes = (16, 24, 24)
    ids = grid_ids(g, 50, 3, torch.int64, 60)
    x, dy = randn(g, 2, 3, 50, 64), randn(g, 2, 3, 50, 64)
    dx = ops().rope_axes(dy, ids, axes, inverse=True)
    for k in range(3):
        d = randn(g, 2, 3, 50, 64)
        up, down = ops().rope_axes(x + d, ids, axes), ops().rope_axes(x - d, ids, axes)
        num = ((up.double() - down.double()) / 2 * dy.double()).sum().item()
        got = (dx.double() * d.double()).sum().item()
        # each rotated value is off by at most 4 * 2^-23 * (|a| + |b|) + u: summed over 19200 terms of size about 1
        assert abs(num - got) <= 19200 * 2.0 ** -20


def test_rope_matches_the_tables():
    """The same rotation as the stepper's cos/sin tables give (model.rope_tables), to the bound of one fp32 rotation."""
    from selas_b200 import model

    g = gen(5)
    axes, l = (16, 56, 56), 77
    ids = grid_ids(g, l, 3, F32, 64)
    cos, sin = model.rope_tables(ids, axes, 10000.0)
    x = randn(g, 1, 2, l, 128)
    a, b = x[..., 0::2], x[..., 1::2]
    tab = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    mag = (a.abs() + b.abs()).repeat_interleave(2, -1)
    assert ((ops().rope_axes(x, ids, axes) - tab).abs() <= 8 * 2.0 ** -23 * mag).all()


def test_rope_not_finite_positions_stay_in_their_token():
    g = gen(6)
    x = randn(g, 1, 2, 4, 8, dtype=BF16)
    ids = torch.tensor([[1.0], [float("inf")], [float("nan")], [3.0]], device=DEV)
    got = ops().rope_axes(x, ids, (8,))
    assert got[:, :, 1:3].isnan().all()
    check_rope(got[:, :, 0::3].contiguous(), x[:, :, 0::3], ids[0::3], (8,))


# ------------------------------------------------------------------------------------------ layer norm


def norm_parts(x, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
    h = c * rstd
    # |error of the kernel's xhat|
    dh = U * (32 * rstd * x.abs().mean(-1, keepdim=True) + 2 * rstd * x.abs() + 24 * h.abs())
    return h, rstd, dh


def check_norm(got, x, w, b, eps):
    h, _, dh = norm_parts(x, eps)
    wf = w.double() if w is not None else torch.ones(x.shape[-1], dtype=F64, device=DEV)
    bf = b.double() if b is not None else torch.zeros_like(wf)
    ref = h * wf + bf
    check(got, ref, dh * wf.abs() + 3 * U * ((h * wf).abs() + bf.abs()), f"norm {tuple(x.shape)}")


DIMS = [1, 2, 3, 4, 7, 8, 16, 24, 31, 32, 33, 63, 64, 65, 96, 100, 127, 128, 129, 256, 384, 511, 512, 513, 640, 768, 896, 1000, 1024, 1025, 1152, 1280, 1536, 1792,
        2047, 2048, 2304, 2560, 3072, 3584, 4096, 4100, 4608, 5120, 6144, 7168,
        8191, 8192, 10240, 12288, 16384, 16385, 20004]


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
def test_norm_sizes(dim, xt):
    g = gen(10)
    for rows in (1, 2, 9, 77, 1500 if dim < 1300 else 400):
        x = randn(g, rows, dim, mean=0.3, dtype=xt)
        w, b = randn(g, dim, std=0.3, mean=1.0), randn(g, dim, std=0.3)
        check_norm(ops().layer_norm(x, w, b), x, w, b, 1e-5)


@pytest.mark.parametrize("xt", [F32, BF16, F16])
@pytest.mark.parametrize("yt", [F32, BF16, F16])
@pytest.mark.parametrize("wt", [F32, BF16, F16])
def test_norm_types(xt, yt, wt):
    g = gen(11)
    for dim in (64, 77, 768, 20004):
        x = randn(g, 13, dim, dtype=xt, std=2.0, mean=-1.0)
        w, b = randn(g, dim, std=0.3, mean=1.0, dtype=wt), randn(g, dim, std=0.3, dtype=wt)
        for wi, bi in ((w, b), (w, None), (None, b), (None, None)):
            got = ops().layer_norm(x, wi, bi, 1e-6, out_dtype=yt)
            assert got.dtype == yt
            check_norm(got, x, wi, bi, 1e-6)


def test_norm_strides():
    """The image rows of a joined [txt | img] stream, rows off a vector's alignment, rows with a stride of their own, one
    dim, many dims, one row for all."""
    g = gen(12)
    x = randn(g, 3, 50, 96)
    w, b = randn(g, 96, mean=1.0), randn(g, 96)
    for v in (x[:, 17:], x[:, ::2], x[..., 1:90], x[:, 3:4], x[1:2], x[0, 0], x.view(3, 5, 10, 96), x[:1, :1].expand(4, 6, 96),
              x.transpose(0, 1), torch.cat((x.flatten(), x[0, 0, :1]))[1:].view(3, 50, 96)):
        d = v.shape[-1]
        check_norm(ops().layer_norm(v, w[:d].clone(), b[:d].clone()), v, w[:d], b[:d], 1e-5)


def test_norm_many_dims_with_a_dim_of_one():
    """Contiguous tensors of four and five dims whose dim of one has some other stride, forward and backward."""
    g = gen(14)
    w, b = randn(g, 96, mean=1.0), randn(g, 96)
    for x in (randn(g, 4, 6, 1, 96).transpose(1, 2), randn(g, 6, 1, 1, 96).transpose(0, 2), randn(g, 5, 2, 1, 3, 96).transpose(1, 2)):
        assert x.is_contiguous()
        check_norm(ops().layer_norm(x, w, b), x, w, b, 1e-5)
        dy = randn(g, *x.shape)
        check_grads(ops().layer_norm_backward(dy, x, w, add=x), grad_ref(dy, x, w.double(), 1e-5, x, False))


def test_norm_hard_rows():
    """A large mean, constant rows, tiny and large values; a row that is not finite stays alone."""
    g = gen(13)
    x = randn(g, 8, 640)
    x[0] += 3000.0
    x[1] = 7.5
    x[2] = 0.0
    x[3] *= 1e-18
    x[4] *= 1e15
    x[5, 3] = 1e4
    w, b = randn(g, 640, mean=1.0), randn(g, 640)
    check_norm(ops().layer_norm(x, w, b), x, w, b, 1e-5)
    y = x.clone()
    y[6, 100] = float("inf")
    y[7, 5] = float("nan")
    got = ops().layer_norm(y, w, b)
    assert got[6:].isnan().all() and torch.equal(got[:6], ops().layer_norm(x, w, b)[:6])


def grad_ref(dy, x, wf, eps, add, per_image):
    """(dx, dw, db) in 64 bits and the bounds of the kernel's errors. wf [.., D] as it multiplies."""
    h, rstd, dh = norm_parts(x, eps)
    dy = dy.double()
    g = dy * wf
    mg, mh = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - mg - h * mh)
    mag = g.abs() + g.abs().mean(-1, keepdim=True) + h.abs() * (g * h).abs().mean(-1, keepdim=True)
    dmh = (g.abs() * dh).mean(-1, keepdim=True) + 40 * U * (g * h).abs().mean(-1, keepdim=True)
    e = rstd * (4 * U * g.abs() + 40 * U * g.abs().mean(-1, keepdim=True) + dh * mh.abs() + h.abs() * dmh + 32 * U * mag)
    ad = add.double() if add is not None else torch.zeros_like(dx)
    e = e + 2 * U * (dx.abs() + ad.abs())
    lead = tuple(range(dy.dim() - 1))
    over = lead[1:] if per_image else lead
    groups = dy.shape[0] if per_image else 1
    rows = dy[..., 0].numel() // max(groups, 1)
    depth = (rows * groups / 296 + 64) if x.shape[-1] <= 16384 else rows / 8 + 64  # roundings in a chain of the sums
    dw, db = (dy * h).sum(over), dy.sum(over)
    ew = (dy.abs() * dh).sum(over) + (depth + 4) * U * (dy * h).abs().sum(over)
    eb = depth * U * dy.abs().sum(over)
    return (dx + ad, e), (dw, ew), (db, eb)


def check_grads(got, refs):
    for name, t, (ref, bound) in zip(("dx", "dw", "db"), got, refs):
        check(t, ref, bound, name)


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
def test_norm_backward_sizes(dim, xt):
    g = gen(20)
    for rows in (1, 3, 77, 1500 if dim < 1300 else 400):
        x, dy = randn(g, rows, dim, mean=0.3, dtype=xt), randn(g, rows, dim, dtype=xt)
        w = randn(g, dim, std=0.3, mean=1.0)
        got = ops().layer_norm_backward(dy, x, w)
        assert got[1].dtype == got[2].dtype == F32
        check_grads(got, grad_ref(dy, x, w.double(), 1e-5, None, False))


@pytest.mark.parametrize("dim", [8, 64, 100, 250, 768, 1000, 2049, 3072, 6144, 12288, 16384])
def test_norm_backward_few_rows(dim):
    """Sums of two rows to many, of one image and of several: one block, the blocks of a cluster, a partial row of sums per
    block. Without the sums dx has the same bits."""
    g = gen(23)
    for b, l in ((1, 2), (1, 5), (1, 9), (1, 20), (1, 33), (1, 64), (1, 129), (1, 260), (2, 7), (5, 13), (9, 8), (9, 20), (17, 40), (40, 3)):
        x, dy = randn(g, b, l, dim, mean=0.3), randn(g, b, l, dim, dtype=BF16)
        s = randn(g, b, dim, std=0.3, dtype=BF16)
        got = ops().ln_mod_backward(dy, x, s)
        ref = grad_ref(dy, x, 1.0 + s.double()[:, None], 1e-6, None, True)
        check_grads((got[0], got[2], got[1]), ref)
        assert torch.equal(ops().ln_mod_backward(dy, x, s, sums=False)[0], got[0])


@pytest.mark.parametrize("xt", [F32, BF16, F16])
@pytest.mark.parametrize("yt", [F32, BF16, F16])
@pytest.mark.parametrize("wt", [F32, BF16, F16, None])
def test_norm_backward_types(xt, yt, wt):
    g = gen(21)
    for dim in (64, 77, 1280, 20004):
        x, dy = randn(g, 2, 31, dim, dtype=xt, std=2.0), randn(g, 2, 31, dim, dtype=yt)
        add = randn(g, 2, 31, dim, dtype=xt)
        w = randn(g, dim, std=0.3, mean=1.0, dtype=wt) if wt else None
        wf = w.double() if wt else torch.ones(dim, dtype=F64, device=DEV)
        for ad in (None, add):
            got = ops().layer_norm_backward(dy, x, w, 1e-6, add=ad)
            assert got[0].dtype == xt
            check_grads(got, grad_ref(dy, x, wf, 1e-6, ad, False))
        dx, dw, db = ops().layer_norm_backward(dy, x, w, 1e-6, add=add, sums=False)
        assert dw is None and db is None and torch.equal(dx, got[0])


def test_norm_backward_strides():
    """Every input with strides of its own (a joined stream's image rows, an expanded dy), and rows off alignment."""
    g = gen(22)
    x, dy, add = randn(g, 3, 50, 96), randn(g, 3, 60, 96, dtype=BF16), randn(g, 3, 33, 100)
    w = randn(g, 96, mean=1.0)
    for vx, vd, va in ((x[:, 17:], dy[:, 5:38], add[..., :96]), (x[:, :33], dy[:1, :1].expand(3, 33, 96), None),
                       (x[:, :33], dy[:, 27:], add[..., 3:99]), (x[..., 1:94][:, :33], dy[:, :33, 2:95], add[..., :93])):
        d = vx.shape[-1]
        wd = w[:d].clone()
        check_grads(ops().layer_norm_backward(vd, vx, wd, add=va), grad_ref(vd, vx, wd.double(), 1e-5, va, False))


@pytest.mark.parametrize("b,l,d", [(1, 1, 64), (1, 300, 3072), (3, 77, 256), (5, 1, 1000), (2, 513, 4100), (400, 3, 128), (2, 9, 16388)])
@pytest.mark.parametrize("yt", [BF16, F32])
def test_mod_backward(b, l, d, yt):
    """Gradients of the adaLN norm, per image; the scale rows as slices of a [B, 6D] modulation, and one row for all."""
    g = gen(23)
    x, dy, add = randn(g, b, l, d, mean=0.2), randn(g, b, l, d, dtype=yt), randn(g, b, l, d)
    mod = randn(g, b, 6 * d, dtype=BF16, std=0.3)
    scale = mod[:, d:2 * d]
    dx, dshift, dscale = ops().ln_mod_backward(dy, x, scale, add=add)
    assert dshift.shape == dscale.shape == (b, d)
    wf = 1 + scale.double()[:, None]
    rx, rw, rb = grad_ref(dy, x, wf, 1e-6, add, True)
    check_grads((dx, dscale, dshift), (rx, rw, rb))
    dx1, dshift1, dscale1 = ops().ln_mod_backward(dy, x, scale[:1])
    assert dshift1.shape == (1, d)
    rx, rw, rb = grad_ref(dy, x, 1 + scale[:1].double()[:, None], 1e-6, None, False)
    check_grads((dx1, dscale1, dshift1), (rx, (rw[0][None], rw[1][None]), (rb[0][None], rb[1][None])))
    assert ops().ln_mod_backward(dy, x, scale, sums=False)[1:] == (None, None)


@pytest.mark.parametrize("dim", [8, 24, 63, 64, 100, 128])
def test_norm_small_rows_eps_zero(dim):
    """Many short rows per warp, the last warp not full, and no eps to hide a division by nothing behind."""
    g = gen(26)
    for rows in (1, 3, 70001):
        x, dy, w = randn(g, rows, dim), randn(g, rows, dim), randn(g, dim, mean=1.0)
        check_norm(ops().layer_norm(x, w, None, 0.0), x, w, None, 0.0)
        check_grads(ops().layer_norm_backward(dy, x, w, 0.0), grad_ref(dy, x, w.double(), 0.0, None, False))


def test_norm_backward_no_rows():
    w = torch.ones(64, device=DEV)
    x = torch.empty(2, 0, 64, device=DEV)
    dx, dw, db = ops().layer_norm_backward(x, x, w)
    assert dx.shape == x.shape and not dw.any() and not db.any() and dw.shape == (64,)
    dx, dsh, dsc = ops().ln_mod_backward(x, x, torch.ones(2, 64, dtype=BF16, device=DEV))
    assert dsh.shape == dsc.shape == (2, 64) and not dsh.any() and not dsc.any()
    e = torch.empty(0, 5, 64, device=DEV)
    assert ops().ln_mod_backward(e, e, torch.ones(0, 64, dtype=BF16, device=DEV))[1].shape == (0, 64)
    assert ops().layer_norm(x, w).shape == x.shape


def test_norm_backward_by_differences():
    """dx, dweight and dbias against central differences of the 64-bit formula of the forward pass."""
    g = gen(24)
    x, dy, w, b = randn(g, 4, 96), randn(g, 4, 96), randn(g, 96, mean=1.0), randn(g, 96)
    dx, dw, db = ops().layer_norm_backward(dy, x, w)

    def loss(x, w, b):
        c = x - x.mean(-1, keepdim=True)
        return ((c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * w + b) * dy.double()).sum().item()

    args, step = (x.double(), w.double(), b.double()), 1e-4
    for n, grad in enumerate((dx, dw, db)):
        for _ in range(3):
            d = randn(g, *args[n].shape).double()
            up, down = ([a + s * step * d if i == n else a for i, a in enumerate(args)] for s in (1, -1))
            num = (loss(*up) - loss(*down)) / (2 * step)
            got = (grad.double() * d).sum().item()
            # the differences' own error is step^2 times the third derivative, below 1e-5 here; 384 terms of 2^-20
            assert abs(num - got) <= 1e-5 * (1 + abs(num)) + 384 * 2.0 ** -20


def test_mod_backward_is_the_gradient_of_ln_mod():
    """Differences of ops.ln_mod itself along large steps of shift and scale, in which it is linear: its bf16 output
    (off by 2^-8 of itself) bounds the comparison."""
    g = gen(25)
    x, dy = randn(g, 2, 40, 256), randn(g, 2, 40, 256, dtype=BF16)
    shift, scale = randn(g, 2, 256, dtype=BF16), randn(g, 2, 256, dtype=BF16, std=0.2)
    _, dsh, dsc = ops().ln_mod_backward(dy, x, scale)
    for n, grad in ((0, dsh), (1, dsc)):
        d = torch.ones(2, 256, dtype=BF16, device=DEV)
        up = ops().ln_mod(x, shift + d * (n == 0), scale + d * (n == 1)).double()
        low = ops().ln_mod(x, shift, scale).double()
        moved = (shift.float() + (n == 0)).to(BF16).double() - shift.double() if n == 0 else (scale.float() + 1).to(BF16).double() - scale.double()
        num = ((up - low) * dy.double()).sum(1)
        tol = ((up.abs() + low.abs()) * 2.0 ** -8 * dy.double().abs()).sum(1) + 1e-3
        assert ((num - grad.double() * moved).abs() <= tol).all()


# ------------------------------------------------------------------------------------------ linear


def act_ref(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "quick_gelu":
        return z * torch.sigmoid(1.702 * z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def check_linear(got, x, w, bias, act, residual, name=""):
    xd, wd = x.double(), w.double()
    z, s = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        z, s = z + bias.double(), s + bias.double().abs()
    y = act_ref(z, act)
    r = residual.double() if residual is not None else torch.zeros_like(y)
    slack = 1.13 * (x.shape[-1] / 16 + 8) * 2.0 ** -22 * s + 8 * U * z.abs() + 2 * U * (y.abs() + r.abs())
    check(got, y + r, slack, name)


def linear_case(g, m, n, k, dt=BF16, bias=True, residual=None):
    x, w = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, std=1 / math.sqrt(max(k, 1)))
    b = randn(g, n, dtype=dt) if bias else None
    r = None if residual is None else randn(g, m, n, dtype=residual)
    return x, w, b, r


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 33, 64, 65, 128, 129, 255, 256, 257, 300, 513, 1030])
def test_linear_rows(m):
    g = gen(30)
    for n, k in ((1, 64), (8, 8), (127, 72), (128, 512), (129, 1000), (700, 2048), (2500, 320)):
        x, w, b, r = linear_case(g, m, n, k, residual=F32)
        check_linear(ops().linear_act(x, w, b, "gelu", r, out_dtype=F32), x, w, b, "gelu", r, f"{m} {n} {k}")
        check_linear(ops().linear_act(x, w), x, w, None, "none", None, f"{m} {n} {k}")


@pytest.mark.parametrize("k", [1, 7, 8, 9, 15, 16, 63, 64, 65, 127, 129, 1001, 4096, 4104])
def test_linear_depths(k):
    """Every K, also where rows do not start on 16 bytes (then copied), one row and one output included."""
    g = gen(31)
    for m, n in ((1, 1), (1, 300), (30, 1), (5, 17), (130, 260), (300, 1111)):
        x, w, b, r = linear_case(g, m, n, k, dt=F16, residual=F16)
        check_linear(ops().linear_act(x, w, b, "silu", r), x, w, b, "silu", r, f"{m} {n} {k}")


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "quick_gelu", "silu"])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_linear_activations_and_types(act, dt):
    g = gen(32)
    for m, n, k in ((3, 200, 256), (140, 132, 192), (600, 520, 128)):
        for bias in (False, True):
            for res in (None, dt, F32):
                for out in (dt, F32):
                    x, w, b, r = linear_case(g, m, n, k, dt, bias, res)
                    got = ops().linear_act(x, w, b, act, r, out_dtype=out)
                    assert got.dtype == out
                    check_linear(got, x, w, b, act, r, f"{m} {bias} {res} {out}")


def test_linear_large_activations():
    """Pre-activations far out on both sides, where exp overflows or an activation is flat."""
    g = gen(33)
    x, w = randn(g, 20, 64, dtype=BF16, std=40.0), randn(g, 72, 64, dtype=BF16)
    for act in ("relu", "gelu", "gelu_tanh", "quick_gelu", "silu"):
        check_linear(ops().linear_act(x, w, None, act, out_dtype=F32), x, w, None, act, None, act)


def test_linear_strides():
    """Row strides, columns of a wider input, a transposed weight, broadcast residual, leading dims, misaligned starts."""
    g = gen(34)
    wide, w, b = randn(g, 40, 400, dtype=BF16), randn(g, 96, 128, dtype=BF16, std=0.1), randn(g, 96, dtype=BF16)
    for x in (wide[:, :128], wide[:, 8:136], wide[:, 3:131], wide[::3, 16:144], wide[5:6, 1:129], wide[:1, :128].expand(9, 128)):
        check_linear(ops().linear_act(x, w, b, "relu"), x, w, b, "relu", None)
    wt = randn(g, 128, 96, dtype=BF16, std=0.1).t()
    x = wide[:, :128]
    check_linear(ops().linear_act(x, wt, b), x, wt, b, "none", None)
    ws = randn(g, 96, 300, dtype=BF16, std=0.1)[:, 5:133]
    check_linear(ops().linear_act(x, ws, b), x, ws, b, "none", None)
    r = randn(g, 1, 96).expand(40, 96)
    check_linear(ops().linear_act(x, w, b, residual=r, out_dtype=F32), x, w, b, "none", r)
    rs = randn(g, 40, 200)[:, 7:103]
    check_linear(ops().linear_act(x, w, b, residual=rs), x, w, b, "none", rs)
    x3 = randn(g, 2, 5, 7, 128, dtype=BF16)
    got = ops().linear_act(x3[:, :, 2:], w, b)
    assert got.shape == (2, 5, 5, 96)
    check_linear(got.reshape(-1, 96), x3[:, :, 2:].reshape(-1, 128), w, b, "none", None)
    x1 = randn(g, 128, dtype=BF16)
    assert torch.equal(ops().linear_act(x1, w, b), ops().linear_act(x1[None], w, b)[0])


@pytest.mark.parametrize("m,n", [(3, 50), (200, 50), (700, 4000)])
def test_linear_no_depth_is_bias_and_residual(m, n):
    b, r = torch.linspace(-2, 2, n, device=DEV).to(BF16), torch.ones(m, n, device=DEV)
    got = ops().linear_act(torch.empty(m, 0, dtype=BF16, device=DEV), torch.empty(n, 0, dtype=BF16, device=DEV), b, "relu", r, out_dtype=F32)
    assert torch.equal(got, b.float().clamp_min(0) + r)


def test_linear_not_finite_stays_in_its_row_and_column():
    g = gen(35)
    for m in (20, 300):
        x, w, b, r = linear_case(g, m, 200, 100, residual=F32)
        clean = ops().linear_act(x, w, b, "none", r)
        x2, w2 = x.clone(), w.clone()
        x2[3, 7] = float("nan")
        w2[50, 99] = float("inf")
        got = ops().linear_act(x2, w2, b, "none", r)
        assert got[3].isnan().all() and not torch.isfinite(got[:, 50]).any()
        keep_r = [i for i in range(m) if i != 3]
        keep_c = [i for i in range(200) if i != 50]
        assert torch.equal(got[keep_r][:, keep_c], clean[keep_r][:, keep_c])
        assert ops().linear_act(x2, w, b, "relu")[3].isnan().all()


def test_linear_writes_only_its_rows():
    """Outputs through the C entry with a row stride of their own: what lies between the rows and after them stays."""
    import ctypes

    from selas_b200 import _lib

    g = gen(36)
    for m, n, k, ld in ((5, 130, 64, 140), (300, 77, 128, 80), (270, 513, 64, 520), (600, 1000, 64, 1003)):
        x, w, b, _ = linear_case(g, m, n, k)
        out = torch.full((m + 1, ld), 7.0, dtype=BF16, device=DEV)
        a = _lib.FbLinearActArgs()
        a.x, a.ldx, a.w, a.ldw, a.bias = x.data_ptr(), k, w.data_ptr(), k, b.data_ptr()
        a.out, a.ld_out, a.m, a.n, a.k = out.data_ptr(), ld, m, n, k
        a.dtype, a.out_dtype, a.act = _lib.FB_BF16, _lib.FB_BF16, _lib.FB_ACT_NONE
        _lib.check(_lib.lib().fb_linear_act(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream), "fb_linear_act")
        check_linear(out[:m, :n], x, w, b, "none", None)
        assert (out[:m, n:] == 7).all() and (out[m] == 7).all()


# ------------------------------------------------------------------------------------------ refusals of the C entries


def test_c_entries_refuse():
    """Bad arguments come back as an error code with a message, and nothing is launched."""
    import ctypes

    from selas_b200 import _lib

    lib = _lib.lib()
    x, y = torch.zeros(2, 64, 64, dtype=BF16, device=DEV)

    def linear(**kw):
        a = _lib.FbLinearActArgs()
        a.x = a.w = a.out = x.data_ptr()
        a.ldx = a.ldw = a.ld_out = 64
        a.m = a.n = a.k = 8
        a.dtype = a.out_dtype = _lib.FB_BF16
        for f, v in kw.items():
            setattr(a, f, v)
        return lib.fb_linear_act(ctypes.addressof(a), None)

    for kw in (dict(m=-1), dict(n=0), dict(k=-1), dict(m=(1 << 30) + 1), dict(n=(1 << 30) + 1), dict(k=(1 << 30) + 1), dict(dtype=_lib.FB_F32), dict(out_dtype=_lib.FB_F16), dict(act=6), dict(x=None),
               dict(out=None), dict(ldx=7), dict(ld_out=4), dict(ldx=9, k=9), dict(out=x.data_ptr() + 1),
               dict(residual=x.data_ptr(), ld_residual=4), dict(residual=x.data_ptr(), ld_residual=8, residual_dtype=_lib.FB_F16)):
        assert linear(**kw) != 0, kw
        assert b"fb_linear_act" in lib.fb_last_error()
    assert lib.fb_linear_act(None, None) != 0

    def norm(fn, **kw):
        a = _lib.FbLayerNormArgs()
        a.x = a.dy = x.data_ptr()
        a.out = y.data_ptr()
        a.outer, a.inner, a.dim = 1, 4, 64
        a.x_inner_stride = a.out_inner_stride = a.dy_inner_stride = 64
        a.x_dtype = a.y_dtype = a.w_dtype = _lib.FB_BF16
        a.eps = 1e-5
        for f, v in kw.items():
            setattr(a, f, v)
        return fn(ctypes.addressof(a), None)

    for fn in (lib.fb_layer_norm, lib.fb_layer_norm_backward):
        for kw in (dict(dim=0), dict(outer=-1), dict(x_dtype=3), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(out=None),
                   dict(x=x.data_ptr() + 1), dict(outer=1 << 20, inner=1 << 20), dict(out=x.data_ptr()), dict(dim=(1 << 30) + 1)):
            assert norm(fn, **kw) != 0, kw
        assert fn(None, None) != 0
    for kw in (dict(dy=None), dict(dy=y.data_ptr()), dict(dweight=x.data_ptr()), dict(dweight=x.data_ptr(), dbias=x.data_ptr(), inner=4000),
               dict(dweight=x.data_ptr(), dbias=x.data_ptr(), outer=70000, inner=1, sum_per_outer=1)):
        assert norm(lib.fb_layer_norm_backward, **kw) != 0, kw

    t = _lib.FbRopeTensor(x.data_ptr(), x.data_ptr(), 64, 64, 64, 64, 64, 64, 1)

    def rope(count=1, dtype=_lib.FB_BF16, batch=1, seq=1, hd=64, ids=x.data_ptr(), idt=0, axes=1, dims=(64,), theta=(1e4,), pairs=0, tensor=t):
        a = _lib.FbRopeArgs()
        a.tensor[0] = a.tensor[1] = tensor
        a.ids, a.ids_stride_l, a.ids_stride_a, a.ids_type = ids, 1, 1, idt
        a.axes_dim[:len(dims)], a.theta[:len(theta)] = dims, theta
        a.count, a.dtype, a.batch, a.seq, a.head_dim, a.axes, a.pairs = count, dtype, batch, seq, hd, axes, pairs
        return lib.fb_rope_axes(ctypes.addressof(a), None)

    for kw in (dict(count=0), dict(count=3), dict(dtype=3), dict(batch=-1), dict(hd=32), dict(ids=None), dict(idt=4), dict(axes=0), dict(axes=9),
               dict(dims=(63,), hd=63), dict(dims=(0,), hd=0), dict(theta=(0.0,)), dict(theta=(float("nan"),)), dict(pairs=2), dict(hd=514, dims=(514,)),
               dict(batch=1 << 16, seq=1 << 16), dict(tensor=_lib.FbRopeTensor(None, x.data_ptr(), 64, 64, 64, 64, 64, 64, 1)),
               dict(tensor=_lib.FbRopeTensor(x.data_ptr(), x.data_ptr(), 64, 64, 64, 64, 64, 64, 0))):
        assert rope(**kw) != 0, kw
    assert lib.fb_rope_axes(None, None) != 0
    torch.cuda.synchronize()
    assert not x.any() and not y.any()


# ------------------------------------------------------------------------------------------ as they are used


def calls(g):
    """One call of each operator at a size that splits its work, and its inputs' refill."""
    x = randn(g, 2, 300, 512)
    dy, scale, mod = randn(g, 2, 300, 512, dtype=BF16), randn(g, 2, 512, dtype=BF16, std=0.2), randn(g, 512, mean=1.0)
    q, ids = randn(g, 2, 4, 300, 128, dtype=BF16), grid_ids(g, 300, 3, torch.int64, 50)
    a, w, b, r = linear_case(g, 20, 700, 2048, residual=F32)
    a2, w2, b2, r2 = linear_case(g, 700, 333, 1001, residual=BF16)  # rows off 16 bytes: through a workspace
    a3, w3, b3, _ = linear_case(g, 4000, 2000, 256)
    return (lambda: ops().layer_norm(x, mod), lambda: ops().layer_norm_backward(dy, x, mod), lambda: ops().ln_mod_backward(dy, x, scale),
            lambda: ops().rope_axes_qk(q, q[:, :2], ids, (16, 56, 56)), lambda: ops().linear_act(a, w, b, "silu", r, out_dtype=F32),
            lambda: ops().linear_act(a2, w2, b2, "gelu", r2), lambda: ops().linear_act(a3, w3, b3, "gelu_tanh"))


def flat(v):
    return [t for u in v for t in flat(u)] if isinstance(v, (list, tuple)) else [v]


def test_same_bits_each_time_and_on_other_streams():
    fs = calls(gen(40))
    first = [flat(f()) for f in fs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for rep in range(3):  # calls of several streams in flight at once
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([flat(f()) for f in fs])
    torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(first, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_and_replayed():
    """Two graphs of the same calls, replayed in turn and with an eager call between, give the eager bits, also after
    their inputs changed."""
    g = gen(41)
    x, dy, w = randn(g, 900, 512), randn(g, 900, 512, dtype=BF16), randn(g, 512, mean=1.0)
    a, wl, b, r = linear_case(g, 24, 512, 1500, residual=F32)
    a2, wl2, _, _ = linear_case(g, 50, 300, 777)

    def step():
        return flat((ops().layer_norm(x, w), ops().layer_norm_backward(dy, x, w, add=x), ops().linear_act(a, wl, b, "gelu", r),
                     ops().linear_act(a2, wl2), ops().rope_axes(x.view(1, 4, 900, 128), torch.arange(900, device=DEV)[:, None], (128,))))

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for k in range(3):
        x.mul_(1.25)
        a.add_(0.5)
        graphs[0][0].replay()
        want = step()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_transformer_layer_from_the_operators():
    """Norm -> projection -> rotary -> attention -> projection + residual -> norm -> MLP with activation -> MLP +
    residual, as a layer of a video or text model would be put together, against the same layer in 64 bits; each
    operator's bf16 output adds 2^-8 relative at most, so the two residual branches stay within 3 % of their norm."""
    g = gen(42)
    b, l, d, h = 2, 200, 512, 4
    axes = (32, 48, 48)
    x = randn(g, b, l, d)
    n1, n2 = (randn(g, d, std=0.1, mean=1.0), randn(g, d, std=0.1)), (randn(g, d, std=0.1, mean=1.0), randn(g, d, std=0.1))
    lin = {k: (randn(g, n, c, dtype=BF16, std=1 / math.sqrt(c)), randn(g, n, dtype=BF16, std=0.1))
           for k, (n, c) in {"qkv": (3 * d, d), "proj": (d, d), "in": (4 * d, d), "out": (d, 4 * d)}.items()}
    ids = torch.stack(torch.meshgrid(torch.arange(2), torch.arange(10), torch.arange(10), indexing="ij"), -1).reshape(-1, 3).to(DEV)
    o = ops()

    y = o.layer_norm(x, *n1, out_dtype=BF16)
    qkv = o.linear_act(y, *lin["qkv"]).view(b, l, 3, h, d // h)
    q, k = o.rope_axes_qk(qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2), ids, axes)
    att = o.attention(q, k, qkv[:, :, 2].transpose(1, 2).contiguous())
    x1 = o.linear_act(att, *lin["proj"], residual=x, out_dtype=F32)
    y = o.layer_norm(x1, *n2, out_dtype=BF16)
    x2 = o.linear_act(o.linear_act(y, *lin["in"], "gelu"), *lin["out"], residual=x1, out_dtype=F32)

    def norm(t, w, bias):
        return torch.nn.functional.layer_norm(t, (d,), w.double(), bias.double(), 1e-5)

    def mm(t, name):
        return t @ lin[name][0].double().t() + lin[name][1].double()

    xd = x.double()
    r = mm(norm(xd, *n1), "qkv").view(b, l, 3, h, d // h)
    rq, rk = (rope_ref(r[:, :, i].transpose(1, 2), ids, axes, 10000.0, "interleaved", False)[0] for i in (0, 1))
    p = torch.softmax(rq @ rk.transpose(-1, -2) / math.sqrt(d // h), -1) @ r[:, :, 2].transpose(1, 2)
    r1 = xd + mm(p.transpose(1, 2).reshape(b, l, d), "proj")
    r2 = r1 + mm(act_ref(mm(norm(r1, *n2), "in"), "gelu"), "out")
    for got, ref, base in ((x1, r1, xd), (x2, r2, xd)):
        assert (got.double() - ref).norm() <= 0.03 * (ref - base).norm()


def test_norm_training_run():
    """A pre-norm residual branch x + f(norm(x)) forward and backward: the gradient that reaches x past the norm is added
    by layer_norm_backward itself; against 64-bit automatic differentiation."""
    g = gen(43)
    d = 384
    x, w, b = randn(g, 3, 50, d), randn(g, d, std=0.2, mean=1.0), randn(g, d, std=0.2)
    m, dy = randn(g, d, d, dtype=BF16, std=1 / math.sqrt(d)), randn(g, 3, 50, d)
    h = ops().layer_norm(x, w, b, out_dtype=BF16)
    y = ops().linear_act(h, m, residual=x, out_dtype=F32)
    dh = (dy.view(-1, d) @ m.float()).view_as(dy)
    dx, dw, db = ops().layer_norm_backward(dh, x, w, add=dy)
    leaves = [t.double().requires_grad_(True) for t in (x, w, b)]
    hn = torch.nn.functional.layer_norm(leaves[0], (d,), leaves[1], leaves[2], 1e-5)
    ref = leaves[0] + hn @ m.double().t()
    want = torch.autograd.grad(ref, leaves, dy.double())
    # h was rounded to bf16 (2^-9 of each value at random): 384 of them average out in y; dh is a plain fp32 product
    assert (y.double() - ref).norm() <= 2.0 ** -8 * (ref - leaves[0]).norm()
    for got, wnt in zip((dx, dw, db), want):
        assert (got.double() - wnt).norm() <= 1e-5 * wnt.norm()
