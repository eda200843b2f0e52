"""Every launch shape of the expert-segment products, at long sums, to the last bit.

Operands are +-1 and +-2, so that each product counts, every partial sum is a whole number far below 2^24, and fp32 sums
are exact in any order: a product that is lost, taken twice or taken from another row changes the result.  The kernel that
a call launches, and the CTAs that share a tile's sum, are read from a captured graph's node.
"""
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

from tests.conftest import cuda_ok  # noqa: E402

if not cuda_ok():
    pytest.skip("needs an sm_100 GPU", allow_module_level=True)
driver = pytest.importorskip("cuda.bindings.driver")

from td_benchmark_b200 import ops  # noqa: E402

DEV = torch.device("cuda", 0)
# rows of a tile, CTA pairs, shared sums, stages, CTAs on an SM
SHAPES = {(256, 1, 0, 6, 1): "wide", (256, 0, 0, 4, 1): "slim", (32, 0, 0, 4, 2): "narrow", (32, 0, 0, 9, 1): "single",
          (32, 0, 1, 4, 2): "split", (64, 0, 1, 7, 1): "split64"}


def _grid(*shape, seed, dtype):
    v = torch.tensor([-2, -1, 1, 2], dtype=torch.int8)
    return v[torch.randint(0, 4, shape, generator=torch.Generator().manual_seed(seed))].to(dtype).to(DEV)


def _ends(counts):
    return torch.tensor(counts, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


def _spans(counts):
    at = 0
    for e, c in enumerate(counts):
        yield e, slice(at, at + c)
        at += c


def _launched(call):
    """(shape, CTAs of a cluster) of the one kernel that the call launches."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        held = call()
    raw = driver.CUgraph(graph.raw_cuda_graph())

    def ok(result):
        assert result[0] == driver.CUresult.CUDA_SUCCESS, result
        return result[1:]

    nodes = ok(driver.cuGraphGetNodes(raw, ok(driver.cuGraphGetNodes(raw, 0))[-1]))[0]
    found = []
    for node in nodes:
        if ok(driver.cuGraphNodeGetType(node))[0] != driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        (params,) = ok(driver.cuGraphKernelNodeGetParams(node))
        name = ok(driver.cuFuncGetName(params.func) if int(params.func) else driver.cuKernelGetName(params.kern))[0]
        shape = re.search(r"grouped_kernel.*ShapeILi(\d+)ELb(\d)ELb(\d)ELi(\d+)ELi(\d+)E", name.decode())
        (cluster,) = ok(driver.cuGraphKernelNodeGetAttribute(
            node, driver.CUlaunchAttributeID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION))
        if shape:
            found.append((SHAPES[tuple(map(int, shape.groups()))], max(1, cluster.clusterDim.x)))
    del held
    assert len(found) == 1, found
    return found[0]


def _exact(got, want):
    """One rounding of whole numbers to the output's type."""
    assert torch.equal(got, want.to(got.dtype)), (got.double() - want).abs().max()


TYPES = [torch.bfloat16, torch.float16]
# (rows of each segment, rows behind them, output columns, summed axis, shape, CTAs that share a sum)
ROWS = [
    ([300, 0, 65, 129], 5, 520, 4104, "split64", 2),
    ([260, 0, 70, 129], 0, 513, 2056, "split64", 2),
    ([257, 1, 63, 64, 0, 190], 9, 264, 4104, "split64", 2),
    ([500], 0, 520, 2056, "split64", 2),
    ([700, 513, 0, 31], 4, 136, 2056, "split64", 2),
    ([3, 0, 9], 3, 264, 4104, "split", 8),
    ([3, 0, 9], 3, 2056, 4104, "split", 4),
    ([30], 2, 1032, 4104, "split", 8),
    ([300, 0, 65, 129], 5, 264, 4104, "split", 4),
    ([1], 0, 4104, 1032, "split", 2),
    ([20, 0, 3, 8], 0, 2056, 4104, "single", 1),
    ([2] * 40, 3, 264, 4104, "single", 1),
    ([2] * 40, 3, 520, 4104, "narrow", 1),
    ([1] * 200 + [13], 7, 264, 2056, "narrow", 1),
    ([700, 513, 0, 31], 4, 520, 4104, "wide", 2),
    ([2100, 1, 700], 5, 1032, 4104, "wide", 2),
    ([64, 128, 256, 63, 65, 255], 40, 2056, 4104, "wide", 2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,slack,cols,summed,shape,parts", ROWS)
def test_rows_times_weights(counts, slack, cols, summed, shape, parts, dtype):
    """The product (weights read along the sum) and the gradient of the rows (read across it), to fp32 and 16 bits."""
    rows, ends = sum(counts) + slack, _ends(counts)
    pad = (summed + 7) // 8 * 8
    x = _grid(rows, summed, seed=1, dtype=dtype)
    for name, product, w in [
            ("forward", ops.grouped_mm, _grid(len(counts), cols, pad, seed=2, dtype=dtype)),
            ("dx", ops.grouped_mm_dx, _grid(len(counts), pad, (cols + 7) // 8 * 8, seed=3, dtype=dtype)[..., :cols])]:
        status = ops.new_status(DEV)
        assert _launched(lambda: product(x, w, ends)) == (shape, parts), name
        want = torch.zeros((rows, cols), dtype=torch.float64, device=DEV)
        for e, s in _spans(counts):
            want[s] = x[s].double() @ (w[e].double().T if name == "forward" else w[e].double())
        _exact(product(x, w, ends, out_dtype=torch.float32, status=status), want)
        _exact(product(x, w, ends, status=status), want)
        out = torch.full((rows, cols), -7.0, device=DEV, dtype=dtype)
        product(x, w, ends, out=out, status=status)
        _exact(out[:rows - slack], want[:rows - slack])
        assert (out[rows - slack:] == -7).all()
        ops.check_status(status)


# (rows of each segment, rows behind them, N, K, shape, CTAs that share a sum)
WEIGHTS = [
    ([8191, 300], 3, 264, 136, "split64", 4), ([8191, 300], 3, 136, 72, "split64", 8), ([9000], 0, 136, 2056, "split64", 2),
    ([0, 4097, 0, 4100], 2, 72, 136, "split64", 8), ([5000, 1], 0, 520, 264, "split64", 2),
    ([2100, 1, 700], 5, 136, 72, "slim", 1), ([64, 128, 0, 63, 65, 4100], 40, 520, 128, "slim", 1),
    ([4111, 1, 700, 0, 64, 65], 5, 520, 264, "wide", 2), ([4111, 1, 700], 5, 1032, 2056, "wide", 2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,slack,n,k,shape,parts", WEIGHTS)
def test_weight_gradients(counts, slack, n, k, shape, parts, dtype):
    rows, ends = sum(counts) + slack, _ends(counts)
    dy, x = _grid(rows, n, seed=1, dtype=dtype), _grid(rows, k, seed=2, dtype=dtype)
    status = ops.new_status(DEV)
    assert _launched(lambda: ops.grouped_mm_dw(dy, x, ends)) == (shape, parts)
    want = torch.stack([dy[s].double().T @ x[s].double() for _, s in _spans(counts)])
    _exact(ops.grouped_mm_dw(dy, x, ends, out_dtype=torch.float32, status=status), want)
    _exact(ops.grouped_mm_dw(dy, x, ends, status=status), want)
    ops.check_status(status)


# (rows of each segment, rows behind them, N, K, shape, CTAs that share a sum)
INTEGERS = [
    ([300, 0, 65, 129], 5, 520, 4112, "split64", 2), ([257, 1, 63, 64, 0, 190], 9, 264, 4112, "split64", 2),
    ([3, 0, 9], 3, 264, 4112, "split", 8), ([30], 2, 2056, 4112, "split", 4), ([300, 0, 65, 129], 5, 136, 2064, "split", 2),
    ([20, 0, 3, 8], 0, 2056, 4112, "single", 1), ([2] * 40, 3, 520, 4112, "narrow", 1),
    ([700, 513, 0, 31], 4, 520, 4112, "wide", 2),
]


@pytest.mark.parametrize("counts,slack,n,k,shape,parts", INTEGERS)
def test_integer_products(counts, slack, n, k, shape, parts):
    rows, ends = sum(counts) + slack, _ends(counts)
    g = torch.Generator().manual_seed(3)
    a = torch.randint(-128, 128, (rows, k), generator=g, dtype=torch.int8).to(DEV)
    w = torch.randint(-128, 128, (len(counts), n, k), generator=g, dtype=torch.int8).to(DEV)
    sa, sw = (torch.rand(rows, generator=g) + 0.5).to(DEV), (torch.rand(len(counts), n, generator=g) + 0.5).to(DEV)
    call = lambda **kw: ops.int8_grouped_mm(a, sa, w, sw, ends, **kw)  # noqa: E731
    assert _launched(call) == (shape, parts)
    want = torch.zeros((rows, n), device=DEV)
    for e, s in _spans(counts):
        want[s] = (a[s].double() @ w[e].double().T).float() * sa[s, None] * sw[e]
    status = ops.new_status(DEV)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(call(out_dtype=dtype, status=status), want.to(dtype))
    ops.check_status(status)
