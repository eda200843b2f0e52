"""What the calls of the expert-segment and integer products pass on, refuse and leave alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from tests.conftest import cuda_ok  # noqa: E402

if not cuda_ok():
    pytest.skip("needs an sm_100 GPU", allow_module_level=True)

import torch.autograd.forward_ad as forward_ad  # noqa: E402

from td_benchmark_b200 import ops  # noqa: E402

DEV = torch.device("cuda", 0)


def _randn(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _ends(counts):
    return torch.tensor(counts, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


@pytest.fixture()
def launches(monkeypatch):
    """(entry, status pointer) of every launch; the status is the last argument before the stream."""
    seen, launch = [], ops._launch
    monkeypatch.setattr(ops, "_launch",
                        lambda device, name, *args: seen.append((name, args[-1])) or launch(device, name, *args))
    return seen


# ---------------------------------------------------------------- status words
def test_status_reaches_every_entry(launches):
    x, w, ends, dy = _randn(6, 64), _randn(2, 32, 64, seed=1), _ends([4, 2]), _randn(6, 32, seed=2)
    status = ops.new_status(DEV)
    q, s = ops.quant_int8(x, status=status)
    wq, sw = ops.quant_int8(w.view(-1, 64), status=status)
    ops.grouped_mm(x, w, ends, status=status)
    ops.grouped_mm_dx(dy, w, ends, status=status)
    ops.grouped_mm_dw(dy, x, ends, status=status)
    ops.int8_mm(q, s, wq, sw, status=status)
    ops.int8_grouped_mm(q, s, wq.view(2, 32, 64), sw.view(2, 32), ends, status=status)
    assert len(launches) == 7 and all(at == status.data_ptr() for _, at in launches), launches
    ops.check_status(status)
    with pytest.raises(ValueError, match="status"):
        ops.int8_mm(q, s, wq, sw, status=torch.zeros(1, device=DEV))


def test_status_of_the_forward_reaches_the_backward(launches):
    x, w = _randn(6, 64).requires_grad_(), _randn(2, 32, 64, seed=1).requires_grad_()
    status = ops.new_status(DEV)
    y = ops.grouped_mm(x, w, _ends([4, 2]), status=status)
    y.backward(torch.ones_like(y))
    assert [name for name, _ in launches] == ["b2m_grouped_mm", "b2m_grouped_mm_dx", "b2m_grouped_mm_dw"]
    assert all(at == status.data_ptr() for _, at in launches)
    ops.check_status(status)
    # ends that are out of order by the time of the backward pass: what it finds is recorded
    ends = _ends([4, 2])
    y = ops.grouped_mm(x, w, ends, status=status)
    ends.data.copy_(torch.tensor([7, 6]))
    y.backward(torch.ones_like(y))
    with pytest.raises(RuntimeError, match="BAD_ROUTING"):
        ops.check_status(status)


# ---------------------------------------------------------------- derivatives that a call would drop
def _all_calls():
    """name -> (call of its float inputs and out, those inputs, an output)."""
    x, w, ends, dy = _randn(6, 64), _randn(2, 32, 64, seed=1), _ends([4, 2]), _randn(6, 32, seed=2)
    q, s = ops.quant_int8(x)
    wq, sw = ops.quant_int8(w.view(-1, 64))
    w3, sw3 = wq.view(2, 32, 64), sw.view(2, 32)
    new = lambda *shape: torch.empty(shape, device=DEV, dtype=torch.bfloat16)  # noqa: E731
    return {
        "grouped_mm_dx": (lambda a, b, o=None: ops.grouped_mm_dx(a, b, ends, out=o), (dy, w), new(6, 64)),
        "grouped_mm_dw": (lambda a, b, o=None: ops.grouped_mm_dw(a, b, ends, out=o), (dy, x), new(2, 32, 64)),
        "quant_int8": (lambda a, o=None: ops.quant_int8(a, scale=o)[1], (x,), torch.empty(6, device=DEV)),
        "int8_mm": (lambda a, b, o=None: ops.int8_mm(q, a, wq, b, out=o), (s, sw), new(6, 64)),
        "int8_grouped_mm": (lambda a, b, o=None: ops.int8_grouped_mm(q, a, w3, b, ends, out=o), (s, sw3), new(6, 32)),
        "grouped_mm": (lambda a, b, o=None: ops.grouped_mm(a, b, ends, out=o), (x, w), new(6, 32)),
    }


NAMES = ["grouped_mm_dx", "grouped_mm_dw", "quant_int8", "int8_mm", "int8_grouped_mm", "grouped_mm"]


@pytest.mark.parametrize("name", NAMES)
def test_gradients_are_not_dropped(name):
    call, inputs, out = _all_calls()[name]
    want = call(*inputs)
    for i in range(len(inputs)):
        held = [t.detach().clone().requires_grad_(i == j) for j, t in enumerate(inputs)]
        if name == "grouped_mm":
            assert call(*held).requires_grad
        else:
            with pytest.raises(ValueError, match=f"{name} is not differentiable"):
                call(*held)
            assert torch.equal(call(*(t.detach() for t in held)), want)
        with torch.no_grad():
            got = call(*held)
        assert torch.equal(got, want) and not got.requires_grad
    with pytest.raises(ValueError, match="not differentiable"):
        call(*inputs, out.requires_grad_())
    with torch.no_grad():
        assert torch.equal(call(*inputs, out), want)


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_not_dropped(name):
    call, inputs, out = _all_calls()[name]
    want = call(*inputs)
    with forward_ad.dual_level():
        for i, t in enumerate(inputs):
            dual = [forward_ad.make_dual(u, torch.ones_like(u)) if i == j else u for j, u in enumerate(inputs)]
            with pytest.raises(ValueError, match=f"{name} has no forward-mode derivative"):
                call(*dual)
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            call(*inputs, forward_ad.make_dual(out, torch.ones_like(out)))
        assert torch.equal(call(*inputs), want)              # nothing carries a tangent


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_refused(name):
    """Batched and differentiated tensors of torch.func have no memory of their own: every call says so."""
    call, inputs, _ = _all_calls()[name]
    first, rest = inputs[0], inputs[1:]
    total = lambda t: call(t, *rest).float().sum()  # noqa: E731
    for run in (lambda: torch.func.vmap(lambda t: call(t, *rest))(first[None]), lambda: torch.func.grad(total)(first),
                lambda: torch.func.jvp(total, (first,), (first,))):
        with pytest.raises((RuntimeError, ValueError)):
            run()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.filterwarnings("ignore::DeprecationWarning", "ignore::torch.jit.TracerWarning")
def test_traces_are_refused(name):
    """A recorded graph would hold an allocation that nothing writes to."""
    from torch.fx.experimental.proxy_tensor import make_fx

    call, inputs, _ = _all_calls()[name]
    one = lambda t: call(t, *inputs[1:])  # noqa: E731
    for record in (lambda: torch.jit.trace(one, inputs[0], check_trace=False), lambda: make_fx(one)(inputs[0]),
                   lambda: make_fx(one, tracing_mode="fake")(inputs[0])):
        with pytest.raises(RuntimeError, match="trace|data pointer"):
            record()


def test_compiled_callers_and_dispatch_modes_work():
    """torch.compile leaves the calls out of its graphs, and modes that only watch do not matter."""
    from torch.utils.flop_counter import FlopCounterMode

    call, inputs, _ = _all_calls()["grouped_mm"]
    want = call(*inputs)
    compiled = torch.compile(lambda a, b: call(a * 1, b) * 1, backend="aot_eager")
    assert torch.equal(compiled(*inputs), want)
    with FlopCounterMode(display=False):
        assert torch.equal(call(*inputs), want)
    x = inputs[0].clone().requires_grad_()
    dy = torch.ones_like(want)
    assert torch.equal(torch.autograd.grad(compiled(x, inputs[1]), x, dy)[0], torch.autograd.grad(call(x, inputs[1]), x, dy)[0])


# ---------------------------------------------------------------- outputs beside an input
@pytest.mark.parametrize("rows,n,k", [(6, 32, 64), (300, 264, 136), (1, 8, 16)])
def test_outputs_beside_an_input_in_one_buffer(rows, n, k):
    """Columns next to an input's columns are an output like any other; nothing else of the buffer changes."""
    counts = [rows - rows // 3, rows // 3]
    ends, w = _ends(counts), _randn(2, n, k, seed=1)
    buf = torch.full((rows, k + n + 24), 7.0, device=DEV, dtype=torch.bfloat16)
    x, out, dy = buf[:, :k], buf[:, k + 8:k + 8 + n], _randn(rows, n, seed=2)
    x.copy_(_randn(rows, k, seed=3))
    plain, kept = x.clone(), x.clone()
    assert torch.equal(ops.grouped_mm(x, w, ends, out=out), ops.grouped_mm(plain, w, ends))
    assert torch.equal(x, kept) and (buf[:, k:k + 8] == 7).all() and (buf[:, k + 8 + n:] == 7).all()
    # dx beside dy
    both = torch.full((rows, n + k), 7.0, device=DEV, dtype=torch.bfloat16)
    both[:, :n] = dy
    assert torch.equal(ops.grouped_mm_dx(both[:, :n], w, ends, out=both[:, n:]), ops.grouped_mm_dx(dy, w, ends))
    assert torch.equal(both[:, :n], dy)
    for bad in (buf[:, k - 1:k - 1 + n], buf[:, :n]):
        with pytest.raises(ValueError, match="overlaps"):
            ops.grouped_mm(x, w, ends, out=bad)


@pytest.mark.parametrize("rows,n,k", [(6, 32, 64), (300, 264, 144), (1, 8, 16)])
def test_integer_outputs_beside_an_input_in_one_buffer(rows, n, k):
    """Codes beside their rows, and integer products beside the codes."""
    ends, w = _ends([rows - rows // 3, rows // 3]), _randn(2 * n, k, seed=1)
    plain = _randn(rows, k, seed=3)
    want, want_s = ops.quant_int8(plain)
    buf = torch.full((rows, 2 * k + 8), 7.0, device=DEV, dtype=torch.bfloat16)
    buf[:, :k] = plain
    q, s = ops.quant_int8(buf[:, :k], q=buf.view(torch.int8)[:, 2 * k + 16:3 * k + 16])
    assert torch.equal(q, want) and torch.equal(s, want_s) and torch.equal(buf[:, :k], plain)
    wq, sw = ops.quant_int8(w)
    wide = torch.full((rows, k + 4 * n), 5, device=DEV, dtype=torch.int8)
    wide[:, :k] = want
    got = ops.int8_grouped_mm(wide[:, :k], s, wq.view(2, n, k), sw.view(2, n), ends,
                              out=wide[:, k:].view(torch.float32))
    assert torch.equal(got, ops.int8_grouped_mm(want, s, wq.view(2, n, k), sw.view(2, n), ends, out_dtype=torch.float32))
    assert torch.equal(wide[:, :k], want)


# ---------------------------------------------------------------- outputs that a graph has saved
@pytest.mark.parametrize("name", NAMES)
def test_a_graph_notices_that_its_saved_values_were_overwritten(name):
    call, inputs, out = _all_calls()[name]
    v = torch.ones(out.shape, device=DEV, dtype=out.dtype, requires_grad=True)
    loss = (out * v).sum()                                   # saves out for v's gradient
    loss.backward(retain_graph=True)
    call(*inputs, out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                             # tensors without a version
        kept = torch.empty_like(out)
        assert torch.equal(call(*inputs, kept), out)


def test_codes_count_as_modified_too():
    x = _randn(6, 64)
    q = torch.zeros((6, 64), device=DEV, dtype=torch.int8)
    before = q._version
    ops.quant_int8(x, q=q)
    assert q._version > before


# ---------------------------------------------------------------- saved tensors
@pytest.mark.parametrize("k", [61, 64])
def test_saved_tensors_that_come_back_in_another_layout(k):
    """Hooks that keep saved tensors on the host bring rows back that lie next to each other, whatever they were."""
    counts, n = [4, 0, 9], 40
    x = torch.full((13, 72), float("nan"), device=DEV, dtype=torch.bfloat16)[:, :k]
    w = torch.full((3, n, 72), float("nan"), device=DEV, dtype=torch.bfloat16)[..., :k]
    x.copy_(_randn(13, k)), w.copy_(_randn(3, n, k, seed=1))
    x.requires_grad_(), w.requires_grad_()
    dy = _randn(13, n, seed=2)
    want = torch.autograd.grad(ops.grouped_mm(x, w, _ends(counts)), (x, w), dy)
    with torch.autograd.graph.save_on_cpu():
        y = ops.grouped_mm(x, w, _ends(counts))
    for got, ref in zip(torch.autograd.grad(y, (x, w), dy), want):
        assert torch.equal(got, ref)


# ---------------------------------------------------------------- orders and distances of the experts
def _experts(kind, experts, rows, cols, dtype, fill):
    """[experts, rows, cols] laid out one behind the other with a gap, or row by row between the others."""
    if kind == "gap":
        base = torch.full((experts * (rows * cols + 48),), fill, device=DEV, dtype=dtype)
        return base, base.as_strided((experts, rows, cols), (rows * cols + 48, cols, 1))
    base = torch.full((rows, experts, cols), fill, device=DEV, dtype=dtype)
    return base, base.transpose(0, 1)


@pytest.mark.parametrize("kind", ["gap", "between"])
@pytest.mark.parametrize("counts,n,k", [([4, 0, 2], 32, 64), ([300, 1, 70], 264, 144), ([5, 0, 9], 264, 4112)])
def test_experts_in_another_order(kind, counts, n, k):
    """Weights and their gradients of any expert stride give what contiguous ones give."""
    rows, ends = sum(counts), _ends(counts)
    x, dy, w = _randn(rows, k), _randn(rows, n, seed=1), _randn(3, n, k, seed=2)
    _, wide = _experts(kind, 3, n, k, torch.bfloat16, float("nan"))
    wide.copy_(w)
    assert torch.equal(ops.grouped_mm(x, wide, ends), ops.grouped_mm(x, w, ends))
    assert torch.equal(ops.grouped_mm_dx(dy, wide, ends), ops.grouped_mm_dx(dy, w, ends))
    a, sa = ops.quant_int8(x)
    q, sw = ops.quant_int8(w.view(-1, k))
    _, wide = _experts(kind, 3, n, k, torch.int8, 77)
    wide.copy_(q.view(3, n, k))
    want = ops.int8_grouped_mm(a, sa, q.view(3, n, k), sw.view(3, n), ends)
    assert torch.equal(ops.int8_grouped_mm(a, sa, wide, sw.view(3, n), ends), want)
    for dtype in (torch.bfloat16, torch.float32):
        base, out = _experts(kind, 3, n, k, dtype, 7.0)
        got = ops.grouped_mm_dw(dy, x, ends, out=out)
        assert torch.equal(got, ops.grouped_mm_dw(dy, x, ends, out_dtype=dtype))
        out.fill_(7.0)
        assert (base == 7).all()                             # nothing between the experts was written
    xr, wr = x.clone().requires_grad_(), _experts(kind, 3, n, k, torch.bfloat16, 0.0)[1].copy_(w).requires_grad_()
    gx, gw = torch.autograd.grad(ops.grouped_mm(xr, wr, ends), (xr, wr), dy)
    assert torch.equal(gx, ops.grouped_mm_dx(dy, w, ends)) and torch.equal(gw, ops.grouped_mm_dw(dy, x, ends))
