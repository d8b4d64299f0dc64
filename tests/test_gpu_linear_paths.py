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
