"""Which kernel a call of ops.linear_act launches, and that kernel's results. The launches are read from a captured graph, so
a test names the kernel that its sizes are there for and fails when the choice moves away from them."""

from __future__ import annotations

import math
import re

import pytest
import torch

from .conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a B200")]

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
DEV = "cuda"


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


def launches(f):
    """(kernel, template arguments, CTAs per cluster) of the library's kernels that f launches, from a graph that f is
    captured into (and that is not run)."""
    from cuda.bindings import driver as cu

    def ok(r):
        assert r[0] == cu.CUresult.CUDA_SUCCESS, r[0]
        return r[1] if len(r) == 2 else r[1:]

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = f()
    g = cu.CUgraph(graph.raw_cuda_graph())
    n = ok(cu.cuGraphGetNodes(g))[1]
    found = []
    for node in ok(cu.cuGraphGetNodes(g, n))[0]:
        if ok(cu.cuGraphNodeGetType(node)) != cu.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        p = ok(cu.cuGraphKernelNodeGetParams(node))
        name = ok(cu.cuKernelGetName(p.kern) if int(p.kern) else cu.cuFuncGetName(p.func)).decode()
        m = re.search(r"(align_rows_kernel|few_kernel|many_kernel)(?:I((?:L[ib]\d+E)+)E)?", name)
        if m:
            attr = cu.CUlaunchAttributeID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION
            cluster = ok(cu.cuGraphKernelNodeGetAttribute(node, attr)).clusterDim.x
            found.append((m[1], tuple(int(v) for v in re.findall(r"L[ib](\d+)E", m[2] or "")), max(cluster, 1)))
    del out
    return found


@pytest.mark.parametrize("m,n", [(129, 40000), (4096, 4096), (5000, 8200)])
def test_no_depth_needs_no_tensor_map(m, n):
    """K = 0 with enough output tiles for the pair kernel, whose tensor maps are not made without a K: the other kernel
    takes the call, and the result is the activated bias plus the residual."""
    x, w = torch.empty(m, 0, dtype=BF16, device=DEV), torch.empty(n, 0, dtype=BF16, device=DEV)
    b, r = torch.linspace(-2, 2, n, device=DEV).to(BF16), torch.ones(m, n, device=DEV)
    call = lambda: ops().linear_act(x, w, b, "relu", r, out_dtype=F32)  # noqa: E731
    assert [k for k, _, _ in launches(call)] == ["few_kernel"]
    assert torch.equal(call(), b.float().clamp_min(0) + r)
    assert not ops().linear_act(x, w).any()


def act_ref(z, act):
    if act == "relu":
        return torch.where(z < 0, 0.0, z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "quick_gelu":
        return z * torch.sigmoid(1.702 * z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "quick_gelu", "silu"])
@pytest.mark.parametrize("m,n,kernel", [(20, 40, "few_kernel"), (300, 20000, "many_kernel")])
def test_activations_of_infinities(act, m, n, kernel):
    """Pre-activations that are infinite, NaN or far out give what the formula gives: NaN where it is inf * 0 or inf - inf.
    With one value per feature times one the pre-activation is exact. An exp that is off by (2 + 1.2 |x|) 2^-23, a
    division by 2^-22 and an erfc by 1.5e-7 move a result by less than 2^-21 |z|; what __fdividef drops is below 1e-36."""
    vals = torch.tensor([-math.inf, math.inf, math.nan, -1e30, 1e30, -3e4, 3e4, -100, 100, -88.5, 88.5, -30, 30, -9, -5, -3, -1, -0.25, 0, 1, 5], device=DEV)
    x, w = torch.zeros(m, 8, dtype=BF16, device=DEV), torch.zeros(n, 8, dtype=BF16, device=DEV)
    x[:, 0] = 1
    w[:, 0] = vals[torch.arange(n, device=DEV) % len(vals)].to(BF16)
    call = lambda: ops().linear_act(x, w, None, act, out_dtype=F32)  # noqa: E731
    assert [k for k, _, _ in launches(call)] == [kernel]
    got, z = call().double(), w[:, 0].double()
    ref = act_ref(z, act)
    assert torch.equal(got.isnan(), ref.isnan().expand(m, n)), (got[0, :21].tolist(), ref[:21].tolist())
    infinite = lambda t: torch.where(t.isinf(), t.sign(), 0.0)  # noqa: E731
    assert torch.equal(infinite(got), infinite(ref).expand(m, n))
    ok = ref.isfinite()
    assert ((got - ref).abs()[:, ok] <= (z.abs() * 2.0 ** -21 + 1e-36)[ok]).all()


# ------------------------------------------------------------------------------------------ large products
#
# Elementwise bounds, with u = 2^-24 and S the sum of magnitudes |x||w|: an accumulator takes 1024 of K, 16 at a time, each
# step off by at most 2^-22 S; its sum is then added in fp32, one rounding per 1024 of K, and partial sums of a shared K are
# added likewise: (min(K, 1024) / 16 + K / 1024 + 8) 2^-22 S, carried through the activation (slope at most 1.13), which
# itself is off by 2^-21 |z| (see above), and two roundings of the sum with the residual.


def randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


class Product:
    """x [m, k], w [n, k], bias and the sums in 64 bits."""

    def __init__(self, m, n, k, dt, seed=1):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.k, self.dt = k, dt
        self.x, self.w, self.b = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, std=1 / math.sqrt(k)), randn(g, n, dtype=dt)
        self.res = {None: None, dt: randn(g, m, n, dtype=dt), F32: randn(g, m, n)}
        self.z = self.x.double() @ self.w.double().t()
        self.s = self.x.double().abs() @ self.w.double().abs().t()

    def call(self, act="none", bias=True, res=None, out=None):
        return ops().linear_act(self.x, self.w, self.b if bias else None, act, self.res[res], out_dtype=out or self.dt)

    def check(self, got, act="none", bias=True, res=None):
        z, s = (self.z + self.b.double(), self.s + self.b.double().abs()) if bias else (self.z, self.s)
        y = act_ref(z, act)
        r = 0.0 if self.res[res] is None else self.res[res].double()
        ref = y + r
        slack = 1.13 * (min(self.k, 1024) / 16 + self.k / 1024 + 8) * 2.0 ** -22 * s + 2.0 ** -21 * z.abs() + 2.0 ** -23 * (y.abs() + abs(r))
        half = ref.abs() * (torch.finfo(got.dtype).eps / 2) + (2.0 ** -25 if got.dtype == F16 else 0.0)
        assert got.shape == ref.shape and torch.isfinite(got).all()
        worst = ((got.double() - ref).abs() / (slack * (1 + torch.finfo(got.dtype).eps) + half + 1e-36)).max().item()
        assert worst <= 1.0, f"{act} bias={bias} residual={res} out={got.dtype}: {worst:.3f} of the bound"


# (m, n, k), the CTAs that share a tile (2: a pair, each tile by itself; more: pairs that share its K; how many fit at once
# depends on how the GPU's SMs are grouped). Rows and columns past the last whole tile, K past the last whole step, columns
# that are no multiple of four (each output by itself), more tiles than pairs, fewer than pairs.
PERSISTENT = [((2601, 4004, 424), (2,)), ((2601, 4003, 424), (2,)), ((2000, 17000, 100), (2,)), ((1500, 9001, 2100), (2,))]
SHARED = [((500, 1020, 8456), (8,)), ((500, 1019, 8456), (8,)), ((1153, 1000, 3736), (4, 6)), ((1000, 2044, 2104), (4,)), ((130, 4097, 8200), (6, 8))]


@pytest.mark.parametrize("size,ctas", PERSISTENT + SHARED)
@pytest.mark.parametrize("dt", [BF16, F16])
def test_large_products(size, ctas, dt):
    """The pair kernel with every activation, bias, residual and output type."""
    p = Product(*size, dt)
    for code, act in enumerate(("none", "relu", "gelu", "gelu_tanh", "quick_gelu", "silu")):
        (kernel, (a, shared), cluster), = [v for v in launches(lambda: p.call(act)) if v[0] != "align_rows_kernel"]
        assert (kernel, a, bool(shared)) == ("many_kernel", code, ctas[0] > 2) and cluster in ctas
        for bias, res, out in ((True, F32, F32), (False, None, dt), (True, dt, dt), (False, F32, dt), (True, dt, F32), (True, None, F32)):
            got = p.call(act, bias, res, out)
            assert got.dtype == out
            p.check(got, act, bias, res)


@pytest.mark.parametrize("m,n,k,kernel", [(4608, 3072, 3072, "many_kernel"), (256, 5001, 4200, "many_kernel"), (300, 3072, 12288, "many_kernel"),
                                          (4000, 1600, 12288, "many_kernel"), (128, 20000, 1600, "few_kernel"), (60, 20000, 2100, "few_kernel"),
                                          (30, 20000, 4200, "few_kernel"), (16, 20000, 4200, "few_kernel"), (128, 20000, 12288, "few_kernel"),
                                          (20, 3072, 12288, "few_kernel")])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_sums_stay_exact_over_a_long_depth(m, n, k, kernel, dt):
    """The sum's error against its norm does not grow with K. A step of 16 of K truncates the accumulator, on average by half
    of the last of its 24 bits, 2^-24 of its size; the size grows as the square root of the steps, so the 64 steps of 1024 of K
    lose 64 * 2/3 * 2^-24 = 2.5e-6 of their sum at most, the sums of several 1024 add up like their sizes, and adding them
    and rounding the output stay below 2e-7. One accumulator for all of K would lose in proportion to K: 1.3e-5 at 12288 and
    4.4e-6 at 4200 were measured."""
    p = Product(m, n, k, dt)
    call = lambda: p.call(bias=False, out=F32)  # noqa: E731
    assert [v[0] for v in launches(call) if v[0] != "align_rows_kernel"] == [kernel]
    got = call()
    p.check(got, bias=False)
    assert (got.double() - p.z).norm() <= 2.7e-6 * p.z.norm()


LARGE = [(2601, 4004, 424), (2601, 4003, 424), (500, 1020, 8456), (500, 1019, 8456)]


@pytest.mark.parametrize("m,n,k", LARGE)
def test_large_products_write_only_their_rows(m, n, k):
    """Through the C entry, with a row stride of the output's own: what lies between the rows and after the last stays."""
    import ctypes

    from selas_b200 import _lib

    p = Product(m, n, k, BF16)
    for ld in (n + 4, n + 37):
        out = torch.full((m + 3, ld), 7.0, dtype=BF16, device=DEV)
        a = _lib.FbLinearActArgs()
        a.x, a.ldx, a.w, a.ldw, a.bias = p.x.data_ptr(), k, p.w.data_ptr(), k, p.b.data_ptr()
        a.out, a.ld_out, a.m, a.n, a.k = out.data_ptr(), ld, m, n, k
        a.dtype, a.out_dtype, a.act = _lib.FB_BF16, _lib.FB_BF16, _lib.FB_ACT_NONE
        call = lambda: _lib.check(_lib.lib().fb_linear_act(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream), "fb_linear_act")  # noqa: E731
        assert [v[0] for v in launches(call)] == ["many_kernel"]
        call()
        p.check(out[:m, :n])
        assert (out[:m, n:] == 7).all() and (out[m:] == 7).all()


@pytest.mark.parametrize("m,n,k", LARGE)
def test_not_finite_stays_in_its_row_and_column_of_a_large_product(m, n, k):
    p = Product(m, n, k, BF16)
    clean = p.call("none", True, F32)
    p.x[m - 1, 7] = float("nan")
    p.w[n - 2, k - 1] = float("inf")
    got = p.call("none", True, F32)
    assert got[m - 1].isnan().all() and not torch.isfinite(got[:, n - 2]).any()
    rows, cols = torch.arange(m, device=DEV) != m - 1, torch.arange(n, device=DEV) != n - 2
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])


def test_large_products_same_bits_on_streams_and_from_graphs():
    """Several in flight at once on streams of their own, and two captured graphs replayed in turn after an input changed."""
    ps = [Product(*size, BF16) for size in LARGE]
    calls = [lambda p=p: p.call("silu", True, F32, F32) for p in ps]
    first = [f() for f in calls]
    for p, y in zip(ps, first):
        p.check(y, "silu", True, F32)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([f() for f in calls])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in outs for a, b in zip(first, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [f() for f in calls]
        graphs.append((g, out))
    for k in range(3):
        for p in ps:
            p.x.mul_(1.25)
        graphs[0][0].replay()
        want = [f() for f in calls]
        graphs[1][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for _, out in graphs for a, b in zip(out, want))
