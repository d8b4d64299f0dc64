"""CPU checks of the token-wise operators (ops.rope_axes, layer_norm, linear_act and their gradients): what they refuse
before any launch, the C structs' layouts, and the workspace sizes the library asks for."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from selas_b200 import _lib, ops
from selas_b200._lib import FluxB200Error

from .conftest import ROOT

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def built():
    from selas_b200 import build

    build.build()


@pytest.fixture
def no_launch(monkeypatch):
    """CPU tensors pass the device check, and a call that gets as far as a launch fails the test."""
    monkeypatch.setattr(ops, "_cuda", lambda *ts: None)

    def launched(*a, **k):
        raise AssertionError("a call that should be refused was launched")

    monkeypatch.setattr(ops, "_launch", launched)


@pytest.mark.parametrize("struct,name", [(_lib.FbRopeTensor, "fb_rope_tensor"), (_lib.FbRopeArgs, "fb_rope_args"),
                                         (_lib.FbLayerNormArgs, "fb_layer_norm_args"),
                                         (_lib.FbLinearActArgs, "fb_linear_act_args")])
def test_struct_layouts_match_c(tmp_path, struct, name):
    fields = [f[0] for f in struct._fields_]
    src = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "flux_b200.h"}"', "int main(void) {",
             f'  printf("size %zu\\n", sizeof({name}));']
    lines += [f'  printf("{f} %zu\\n", offsetof({name}, {f}));' for f in fields]
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(src)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(struct)
    for f in fields:
        assert int(got[f]) == getattr(struct, f).offset, f


@pytest.mark.parametrize("struct,pack,n", [(_lib.FbRopeArgs, _lib.pack_rope, 47), (_lib.FbLayerNormArgs, _lib.pack_layer_norm, 28),
                                           (_lib.FbLinearActArgs, _lib.pack_linear_act, 18)])
def test_packed_arguments_fill_the_struct(struct, pack, n):
    """Numbers 1..n packed in order land in the fields in order."""
    def leaves(s):
        for name, t in s._fields_:
            v = getattr(s, name)
            if isinstance(v, ctypes.Array):
                for e in v:
                    yield from leaves(e) if isinstance(e, ctypes.Structure) else (e,)
            else:
                yield v

    raw = pack(*range(1, n + 1))
    assert len(raw) == ctypes.sizeof(struct)
    assert [int(v) for v in leaves(struct.from_buffer_copy(raw))] == list(range(1, n + 1))


def test_values_that_no_field_holds_are_refused(no_launch):
    wide = torch.zeros(1, dtype=BF16).expand(1 << 31, 1)
    for call in (lambda: ops.layer_norm(X, eps=1e300), lambda: _lib.pack_linear_act(*(1 << 31,) * 18),
                 lambda: ops.linear_act(torch.zeros(1, 0, dtype=BF16), wide[:, :0])):
        with pytest.raises(FluxB200Error, match="out of range"):
            call()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 8, dtype=BF16), torch.zeros(8, 8, dtype=BF16)
    ids = torch.zeros(2, 1)
    for call in (lambda: ops.rope_axes(x.view(1, 1, 2, 8), ids, (8,)), lambda: ops.layer_norm(x),
                 lambda: ops.layer_norm_backward(x, x), lambda: ops.ln_mod_backward(x[None], x[None].float(), x[:1]),
                 lambda: ops.linear_act(x, w)):
        with pytest.raises(FluxB200Error, match="CUDA"):
            call()


Q = torch.zeros(2, 3, 5, 8, dtype=BF16)
IDS = torch.zeros(5, 2)


@pytest.mark.parametrize("match,call", [
    ("add up", lambda: ops.rope_axes(Q, IDS, (4, 2))),
    ("add up", lambda: ops.rope_axes(Q, IDS[:, :1], (10,))),
    ("ids must be", lambda: ops.rope_axes(Q, IDS[:4], (4, 4))),
    ("ids must be", lambda: ops.rope_axes(Q, IDS[:, :1], (4, 4))),
    ("ids must be", lambda: ops.rope_axes(Q, torch.zeros(3, 5, 2), (4, 4))),
    ("ids must be", lambda: ops.rope_axes(Q, IDS.bool(), (4, 4))),
    ("one base, or one per axis", lambda: ops.rope_axes(Q, IDS, (4, 4), (1e4, 1e4, 1e4))),
    ("pairs", lambda: ops.rope_axes(Q, IDS, (4, 4), pairs="neox")),
    ("fp32, bf16 or fp16", lambda: ops.rope_axes(Q.double(), IDS, (4, 4))),
    ("fp32, bf16 or fp16", lambda: ops.rope_axes(Q[0], IDS, (4, 4))),
    ("unit stride", lambda: ops.rope_axes(torch.zeros(2, 3, 8, 5, dtype=BF16).transpose(2, 3), IDS, (4, 4))),
    ("of one type", lambda: ops.rope_axes_qk(Q, Q.float(), IDS, (4, 4))),
    ("of one type", lambda: ops.rope_axes_qk(Q, Q[:1], IDS, (4, 4))),
])
def test_rope_refuses(no_launch, match, call):
    with pytest.raises(FluxB200Error, match=match):
        call()


X = torch.zeros(2, 5, 8)
W = torch.ones(8)


@pytest.mark.parametrize("match,call", [
    ("fp32, bf16 or fp16", lambda: ops.layer_norm(X.double())),
    ("fp32, bf16 or fp16", lambda: ops.layer_norm(X[:, :, :0])),
    ("weight must be", lambda: ops.layer_norm(X, W[:7])),
    ("weight must be", lambda: ops.layer_norm(X, torch.ones(16)[::2])),
    ("share a type", lambda: ops.layer_norm(X, W, W.bfloat16())),
    ("out_dtype", lambda: ops.layer_norm(X, W, out_dtype=torch.float64)),
    ("unit stride", lambda: ops.layer_norm(torch.zeros(2, 8, 5).transpose(1, 2))),
    ("more than three", lambda: ops.layer_norm(torch.zeros(2, 2, 6, 8)[:, :, :5])),
    ("dy must be", lambda: ops.layer_norm_backward(X[:1], X)),
    ("dy must be", lambda: ops.layer_norm_backward(X.double(), X)),
    ("add must be", lambda: ops.layer_norm_backward(X, X, add=X.bfloat16())),
    ("add must be", lambda: ops.layer_norm_backward(X, X, add=X[:1])),
    ("x must be fp32", lambda: ops.ln_mod_backward(X, X.bfloat16(), torch.zeros(2, 8, dtype=BF16))),
    ("x must be fp32", lambda: ops.ln_mod_backward(X[0], X[0], torch.zeros(1, 8, dtype=BF16))),
    ("must be bf16", lambda: ops.ln_mod_backward(X, X, torch.zeros(2, 8))),
    ("scale must be", lambda: ops.ln_mod_backward(torch.zeros(8, 2, 8), torch.zeros(8, 2, 8), torch.zeros(8, dtype=BF16))),
    ("batch does not match", lambda: ops.ln_mod_backward(X, X, torch.zeros(3, 8, dtype=BF16))),
])
def test_norm_refuses(no_launch, match, call):
    with pytest.raises(FluxB200Error, match=match):
        call()


A, B = torch.zeros(3, 16, dtype=BF16), torch.zeros(8, 16, dtype=BF16)


@pytest.mark.parametrize("match,call", [
    ("both be bf16 or both fp16", lambda: ops.linear_act(A.float(), B.float())),
    ("both be bf16 or both fp16", lambda: ops.linear_act(A, B.half())),
    ("K mismatch", lambda: ops.linear_act(A, B[:, :8])),
    ("act must be", lambda: ops.linear_act(A, B, act="tanh")),
    ("out_dtype", lambda: ops.linear_act(A, B, out_dtype=F16)),
    ("bias must be", lambda: ops.linear_act(A, B, torch.zeros(8))),
    ("bias must be", lambda: ops.linear_act(A, B, torch.zeros(7, dtype=BF16))),
    ("residual must be", lambda: ops.linear_act(A, B, residual=torch.zeros(3, 8, dtype=F16))),
    ("residual must be", lambda: ops.linear_act(A, B, residual=torch.zeros(2, 8))),
    ("residual must be", lambda: ops.linear_act(A[0], B, residual=torch.zeros(()))),
    ("at least one row", lambda: ops.linear_act(A, B[:0])),
])
def test_linear_act_refuses(no_launch, match, call):
    with pytest.raises(FluxB200Error, match=match):
        call()


def test_no_rows_launch_nothing(no_launch):
    assert ops.layer_norm(X[:0]).shape == (0, 5, 8)
    assert ops.linear_act(A[:0], B).shape == (0, 8)
    assert ops.rope_axes(Q[:, :, :0], IDS[:0], (4, 4)).shape == (2, 3, 0, 8)


def test_norm_workspace_sizes():
    """One partial row of sums per block when a sum has more than one; nothing for one block or no rows."""
    f = _lib.load().fb_layer_norm_work_floats
    assert f(1, 0, 64, 0) == 0 and f(0, 5, 64, 1) == 0
    assert f(1, 1, 3072, 0) == 0
    n = f(1, 4608, 3072, 0)
    assert n > 0 and n % (2 * 3072) == 0
    assert f(4, 1152, 3072, 0) == n  # a shared weight sums over all rows alike
    per = f(4, 1152, 3072, 1)
    assert per % (4 * 2 * 3072) == 0 and per <= n
    assert f(1, 3, 50000, 0) == 2 * 3  # rows too wide for registers: mean and rstd of each


def test_linear_workspace_only_for_rows_off_16_bytes():
    f = _lib.load().fb_linear_act_work_bytes

    def need(m, n, k, ldx, ldw, x=4096, w=4096):
        a = _lib.FbLinearActArgs()
        a.x, a.w, a.ldx, a.ldw, a.m, a.n, a.k = x, w, ldx, ldw, m, n, k
        return f(ctypes.addressof(a))

    assert need(5, 7, 64, 64, 64) == 0
    assert need(5, 7, 63, 64, 72) == 0  # an odd k in padded rows needs no copy
    assert need(5, 7, 63, 63, 64) == 5 * 64 * 2
    assert need(5, 7, 63, 64, 63) == 7 * 64 * 2
    assert need(5, 7, 63, 63, 63) == 12 * 64 * 2
    assert need(1, 7, 63, 63, 64) == 0  # a single row has no stride
    assert need(1, 7, 64, 64, 64, x=4098) == 64 * 2
    assert need(0, 7, 63, 63, 63) == 0 and need(5, 7, 0, 0, 0) == 0


@pytest.mark.parametrize("x", [torch.zeros(4, 6, 1, 8).transpose(1, 2), torch.zeros(4, 1, 6, 8), torch.zeros(6, 1, 1, 8).transpose(0, 2),
                               torch.zeros(2, 3, 5, 8), torch.zeros(5, 2, 1, 3, 8).transpose(1, 2)])
def test_norm_rows_of_many_dims_are_where_torch_has_them(monkeypatch, x):
    """A dim of one may have any stride and leaves a tensor contiguous: the rows the kernels walk over are the tensor's."""
    packed = []
    monkeypatch.setattr(ops, "_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_launch", lambda index, entry, flops, nbytes, args: packed.append(args))
    ops.layer_norm(x)
    ops.layer_norm_backward(x, x, add=x, sums=False)
    want = (torch.arange(x.numel()).view(-1, 8)[:, 0]).tolist()  # contiguous: row r starts at 8 r
    for raw in packed:
        a = _lib.FbLayerNormArgs.from_buffer_copy(raw)
        for outer, inner in ((a.x_outer_stride, a.x_inner_stride), (a.dy_outer_stride, a.dy_inner_stride),
                             (a.add_outer_stride, a.add_inner_stride)) if a.dy else ((a.x_outer_stride, a.x_inner_stride),):
            assert [o * outer + i * inner for o in range(a.outer) for i in range(a.inner)] == want
