"""Products over expert segments and 8-bit integer products against plain sums in 64 bits.

Tolerances.  A 16-bit output is off by its rounding, half a step of the value (``eps / 2``), and by the fp32 sum before
it: each of the L additions of a sum loses at most one part in 2^23 of a partial sum (an adder that cuts off instead of
rounding loses up to a whole step), and no partial sum passes S = sum |x||w|, so L * 2^-23 * S.  Integer sums are exact:
their outputs are those of the three fp32 roundings that the definition names, bit for bit.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

from tests.conftest import cuda_ok  # noqa: E402

if not cuda_ok():
    pytest.skip("needs an sm_100 GPU", allow_module_level=True)

from td_benchmark_b200 import configs, data, ops  # noqa: E402

DEV = torch.device("cuda", 0)
TYPES = [torch.bfloat16, torch.float16]


def _randn(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def _ends(counts):
    return torch.tensor(counts, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


def _spans(counts):
    at = 0
    for e, c in enumerate(counts):
        yield e, slice(at, at + c)
        at += c


def _close(got, want, mass, length):
    """want and mass (the sums of absolute products) in 64 bits; length = products in a sum."""
    assert got.shape == want.shape
    lost = length * 2.0 ** -23 * mass
    # fp16 results below its normal range are rounded to half of its smallest step
    tol = torch.finfo(got.dtype).eps / 2 * (want.abs() + lost) + lost + torch.finfo(got.dtype).smallest_normal * \
        torch.finfo(got.dtype).eps / 2
    worst = ((got.double() - want).abs() - tol).max().item() if got.numel() else -1.0
    assert worst <= 0, f"past the tolerance by {worst}"


def _fwd(x, w, counts):
    y = x.new_zeros((x.shape[0], w.shape[1]), dtype=torch.float64)
    for e, s in _spans(counts):
        y[s] = x[s].double() @ w[e].double().T
    return y


def _dx(dy, w, counts):
    return _fwd(dy, w.transpose(1, 2), counts)


def _dw(dy, x, counts):
    return torch.stack([dy[s].double().T @ x[s].double() for _, s in _spans(counts)])


# (rows of each expert, rows behind them, N, K)
SHAPES = [
    ([1], 0, 8, 8),
    ([1], 0, 128, 64),
    ([16], 3, 256, 72),
    ([0, 0, 5, 0], 0, 136, 16),
    ([7, 0, 300, 17, 0, 1], 11, 200, 328),
    ([33, 257, 0, 31], 0, 520, 136),
    ([513], 1, 304, 1000),
    ([0, 0, 0], 9, 64, 64),
    ([64, 128, 256, 63, 65, 255], 40, 128, 256),
    ([1] * 200 + [0] * 56 + [3] * 10, 2, 264, 192),
    ([2, 0, 0, 1] * 256, 0, 64, 128),
    ([5000, 3, 1200], 5, 640, 704),
    ([700, 0, 41, 3] + [0] * 96, 0, 136, 200),          # short on average, one segment of many tiles
    ([40] * 300, 0, 72, 80),                              # long on average, more segments than are sorted
    ([20, 0] * 512, 7, 16, 64),                           # 1024 experts
    ([257, 513, 1025, 1793, 2049, 256, 512], 0, 264, 96),  # lengths that tiles share evenly
    ([1], 0, 136, 4104), ([2, 0, 9], 3, 4104, 264),        # few tiles: clusters share a tile's sum
    ([33, 0, 0, 2, 5], 4, 520, 1032), ([30], 0, 1032, 2056), ([8], 40, 264, 1000),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,slack,n,k", SHAPES)
def test_products_over_segments(counts, slack, n, k, dtype):
    rows = sum(counts) + slack
    x, dy = _randn(rows, k, seed=1, dtype=dtype), _randn(rows, n, seed=2, dtype=dtype)
    w = _randn(len(counts), n, k, seed=3, dtype=dtype, std=0.1)
    ends = _ends(counts)
    status = ops.new_status(DEV)
    y = ops.grouped_mm(x, w, ends, status=status)
    dx = ops.grouped_mm_dx(dy, w, ends, status=status)
    dw = ops.grouped_mm_dw(dy, x, ends, status=status)
    torch.cuda.synchronize()
    ops.check_status(status)
    _close(y, _fwd(x, w, counts), _fwd(x.abs(), w.abs(), counts), k)
    _close(dx, _dx(dy, w, counts), _dx(dy.abs(), w.abs(), counts), n)
    _close(dw, _dw(dy, x, counts), _dw(dy.abs(), x.abs(), counts), max(counts))
    if slack:
        assert not y[-slack:].any() and not dx[-slack:].any()


@pytest.mark.parametrize("counts,n,k", [([7, 0, 300, 17], 201, 136), ([3, 1], 1, 64), ([40], 127, 24),
                                        ([300, 2], 1025, 104)])
def test_odd_widths_and_fp32_outputs(counts, n, k):
    """N needs no alignment in a product; a summed axis needs it only in its row stride."""
    rows = sum(counts)
    pad = torch.full((rows, k + 8), float("nan"), device=DEV, dtype=torch.bfloat16)
    wide = torch.full((len(counts), n, k + 16), float("nan"), device=DEV, dtype=torch.bfloat16)
    x, w = pad[:, :k - 3], wide[:, :, :k - 3]
    x.copy_(_randn(rows, k - 3, seed=4))
    w.copy_(_randn(len(counts), n, k - 3, seed=5))
    y = ops.grouped_mm(x, w, _ends(counts), out_dtype=torch.float32)
    assert y.dtype == torch.float32
    _close(y, _fwd(x, w, counts), _fwd(x.abs(), w.abs(), counts), k)
    dy = torch.full((rows, (n + 15) // 8 * 8), float("nan"), device=DEV, dtype=torch.bfloat16)[:, :n]
    dy.copy_(_randn(rows, n, seed=6))
    dx = ops.grouped_mm_dx(dy, w, _ends(counts), out_dtype=torch.float32)
    dw = ops.grouped_mm_dw(dy, x, _ends(counts), out_dtype=torch.float32)
    _close(dx, _dx(dy, w, counts), _dx(dy.abs(), w.abs(), counts), n)
    _close(dw, _dw(dy, x, counts), _dw(dy.abs(), x.abs(), counts), max(counts))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_no_expert_enter_nothing(bad):
    """Rows behind the last segment, and another segment's rows, reach no other output whatever they hold."""
    counts, n, k = [5, 70, 0, 129], 136, 200
    rows = sum(counts)
    x, dy = _randn(rows + 30, k, seed=7), _randn(rows + 30, n, seed=8)
    w = _randn(4, n, k, seed=9)
    x[rows:], dy[rows:] = bad, bad
    x[5:75], dy[5:75] = bad, bad            # the second expert's rows
    ends = _ends(counts)
    y, dx, dw = ops.grouped_mm(x, w, ends), ops.grouped_mm_dx(dy, w, ends), ops.grouped_mm_dw(dy, x, ends)
    keep = [0, 2, 3]
    others = torch.cat([torch.arange(5), torch.arange(75, rows + 30)]).to(DEV)
    assert torch.isfinite(y[others]).all() and torch.isfinite(dx[others]).all() and torch.isfinite(dw[keep]).all()
    assert not torch.isfinite(y[5:75]).any() and not torch.isfinite(dw[1]).any()
    clean = [5, 0, 0, 129]
    cx, cdy = torch.cat([x[:5], x[75:rows]]), torch.cat([dy[:5], dy[75:rows]])
    _close(dw[keep], _dw(cdy, cx, clean)[keep], _dw(cdy.abs(), cx.abs(), clean)[keep], 129)
    _close(y[75:rows], _fwd(cx, w, clean)[5:], _fwd(cx.abs(), w.abs(), clean)[5:], k)


def test_given_output_keeps_rows_of_no_expert_and_columns_beside_it():
    counts, n, k = [3, 40], 72, 64
    x, w, ends = _randn(50, k, seed=1), _randn(2, n, k, seed=2), _ends(counts)
    buf = torch.full((50, n + 24), 7.0, device=DEV, dtype=torch.bfloat16)
    out = buf[:, 8:8 + n]
    assert ops.grouped_mm(x, w, ends, out=out) is out
    _close(out[:43], _fwd(x, w, counts)[:43], _fwd(x.abs(), w.abs(), counts)[:43], k)
    assert (buf[43:] == 7).all() and (buf[:, :8] == 7).all() and (buf[:, 8 + n:] == 7).all()
    big = torch.full((2, n, k + 8), 7.0, device=DEV, dtype=torch.float32)
    ops.grouped_mm_dw(_randn(50, n, seed=3), x, ends, out=big[:, :, :k])
    assert (big[:, :, k:] == 7).all() and not (big[:, :, :k] == 7).any()


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5])
@pytest.mark.parametrize("cols,pitch", [(1, 1), (2, 3), (63, 72), (64, 65), (66, 80), (201, 201), (130, 134), (257, 300), (1713, 1713)])
def test_outputs_that_start_anywhere(cols, pitch, offset):
    """Output rows at any element and pitch, and nothing beside them written: 16-bit, fp32 and weight gradients."""
    counts, k = [37, 0, 300, 1], 72
    rows, wide = sum(counts), (cols + 7) // 8 * 8
    x, w, ends = _randn(rows, k), _randn(4, cols, k, seed=1), _ends(counts)
    dy = _randn(rows, wide, seed=2)[:, :cols]
    want, mass = _fwd(x, w, counts), _fwd(x.abs(), w.abs(), counts)
    for dtype in (torch.bfloat16, torch.float32):
        flat = torch.full((offset + rows * pitch + 8,), -7.0, device=DEV, dtype=dtype)
        out = flat.as_strided((rows, cols), (pitch, 1), offset)
        ops.grouped_mm(x, w, ends, out=out)
        _close(out, want, mass, k)
        out.fill_(-7.0)
        assert (flat == -7.0).all()
    flat = torch.full((offset + 4 * k * pitch + 8,), -7.0, device=DEV, dtype=torch.bfloat16)
    out = flat.as_strided((4, k, cols), (k * pitch, pitch, 1), offset)
    ops.grouped_mm_dw(x, dy, ends, out=out)
    _close(out, _dw(x, dy, counts), _dw(x.abs(), dy.abs(), counts), 300)
    out.fill_(-7.0)
    assert (flat == -7.0).all()


@pytest.mark.parametrize("counts", [[63], [64], [65], [129], [191], [193], [257], [385], [1000], [129, 0, 65], [40, 300, 2],
                                    [2100], [5000], [3000, 0, 1, 70, 2500], [0, 6000, 0], [1, 8191]])
@pytest.mark.parametrize("n,k", [(40, 264), (264, 40), (300, 136)])
def test_few_tiles(counts, n, k):
    """Calls of few tiles, whose tiles have fewer rows: one tile and one more or one less than full ones."""
    rows = sum(counts)
    x, w, ends = _randn(rows, k), _randn(len(counts), n, k, seed=1), _ends(counts)
    dy = _randn(rows, (n + 7) // 8 * 8, seed=2)[:, :n]
    _close(ops.grouped_mm(x, w, ends), _fwd(x, w, counts), _fwd(x.abs(), w.abs(), counts), k)
    _close(ops.grouped_mm_dx(dy, w, ends), _dx(dy, w, counts), _dx(dy.abs(), w.abs(), counts), n)
    _close(ops.grouped_mm_dw(dy, x, ends), _dw(dy, x, counts), _dw(dy.abs(), x.abs(), counts), max(counts))


@pytest.mark.parametrize("counts", [[200] * 9, [1, 0, 63, 64, 65, 130], [0] * 40 + [3] * 200, [3000]])
@pytest.mark.parametrize("n,k", [(264, 128), (1000, 64), (2056, 16), (72, 120), (513, 1)])
def test_weight_gradients_of_few_columns(counts, n, k):
    rows = sum(counts)
    dy = _randn(rows, (n + 7) // 8 * 8, seed=1)[:, :n]
    x = _randn(rows, (k + 7) // 8 * 8, seed=2)[:, :k]
    got = ops.grouped_mm_dw(dy, x, _ends(counts))
    _close(got, _dw(dy, x, counts), _dw(dy.abs(), x.abs(), counts), max(counts))


@pytest.mark.parametrize("experts", [31, 32, 33, 255, 256, 257, 400])
def test_many_segments_of_any_length(experts):
    """Walks in order of length: segments of no row, of few, and of several tiles, in any order."""
    g = torch.Generator().manual_seed(experts)
    counts = torch.randint(0, 60, (experts,), generator=g).tolist()
    for e, c in zip(torch.randperm(experts, generator=g)[:8].tolist(), (0, 0, 31, 32, 257, 511, 700, 1300)):
        counts[e] = c
    n, k = 136, 72
    rows = sum(counts) + 5
    x, w, ends = _randn(rows, k), _randn(experts, n, k, seed=1), _ends(counts)
    dy = _randn(rows, n, seed=2)
    _close(ops.grouped_mm(x, w, ends), _fwd(x, w, counts), _fwd(x.abs(), w.abs(), counts), k)
    _close(ops.grouped_mm_dx(dy, w, ends), _dx(dy, w, counts), _dx(dy.abs(), w.abs(), counts), n)
    _close(ops.grouped_mm_dw(x, dy, ends), _dw(x, dy, counts), _dw(x.abs(), dy.abs(), counts), max(counts))


def test_no_rows():
    w, ends = _randn(3, 64, 32, seed=1), _ends([0, 0, 0])
    x, dy = _randn(0, 32), _randn(0, 64)
    assert ops.grouped_mm(x, w, ends).shape == (0, 64) and ops.grouped_mm_dx(dy, w, ends).shape == (0, 32)
    dw = ops.grouped_mm_dw(dy, x, ends, out=torch.full((3, 64, 32), 5.0, device=DEV, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    assert not dw.any()
    q, s = ops.quant_int8(_randn(0, 32))
    assert q.shape == (0, 32) and s.shape == (0,)


def test_ends_out_of_order_are_recorded_and_contained():
    """An end below an earlier one leaves its segment empty, one past the rows ends at the last row."""
    n, k = 64, 64
    x, w = _randn(40, k, seed=1), _randn(4, n, k, seed=2)
    status = ops.new_status(DEV)
    guard = torch.full((60, n), 7.0, device=DEV, dtype=torch.bfloat16)
    ends = torch.tensor([10, 4, -3, 1 << 30], dtype=torch.int32, device=DEV)
    ops.grouped_mm(x, w, ends, out=guard[:40], status=status)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="BAD_ROUTING"):
        ops.check_status(status)
    _close(guard[:40], _fwd(x, w, [10, 0, 0, 30]), _fwd(x.abs(), w.abs(), [10, 0, 0, 30]), k)
    assert (guard[40:] == 7).all()
    for bad in ([-1, 10, 20, 40], [41, 41, 41, 41], [10, 20, 19, 40]):
        status.zero_()
        ops.grouped_mm_dw(_randn(40, n, seed=3), x, torch.tensor(bad, dtype=torch.int32, device=DEV), status=status)
        assert status.item() == 0x201, bad
    status.zero_()
    ops.grouped_mm(x, w, torch.tensor([0, 10, 10, 40], dtype=torch.int32, device=DEV), status=status)
    assert status.item() == 0


def test_offsets_past_32_bits():
    """The last expert's weights, and the last rows, lie more than 2^32 bytes into their tensors."""
    n, k, experts = 4096, 8192, 66
    w = torch.empty((experts, n, k), dtype=torch.bfloat16, device=DEV)      # 4.4 GB
    w[-1] = _randn(n, k, seed=1)
    w[0] = 0
    counts = [2] + [0] * (experts - 2) + [3]
    x = _randn(5, k, seed=2)
    y = ops.grouped_mm(x, w, _ends(counts))
    want = x[2:].double() @ w[-1].double().T
    _close(y[2:], want, x[2:].abs().double() @ w[-1].abs().double().T, k)
    dy = _randn(5, n, seed=3)
    w.zero_()
    dw = ops.grouped_mm_dw(dy, x, _ends(counts), out=w)
    _close(dw[-1], dy[2:].double().T @ x[2:].double(), dy[2:].abs().double().T @ x[2:].abs().double(), 3)
    del w, dw
    rows = (1 << 31) // 512 + 300
    big = torch.zeros((rows, 512), dtype=torch.bfloat16, device=DEV)        # rows past 2^31 elements
    big[-3:] = _randn(3, 512, seed=4)
    w2 = _randn(2, 1024, 512, seed=5)
    y = ops.grouped_mm(big, w2, torch.tensor([rows - 2, rows], dtype=torch.int32, device=DEV))
    _close(y[-2:], big[-2:].double() @ w2[1].double().T, big[-2:].abs().double() @ w2[1].abs().double().T, 512)
    _close(y[-3:-2], big[-3:-2].double() @ w2[0].double().T, big[-3:-2].abs().double() @ w2[0].abs().double().T, 512)


# ---------------------------------------------------------------- gradients
def test_gradients_through_autograd():
    """The gradients that torch sees are the formula's, with an expanded, a transposed and a ragged-width dy."""
    counts, k = [4, 0, 90, 33], 72
    rows = sum(counts) + 6
    for n, shape in [(64, "plain"), (64, "transposed"), (64, "expanded"), (61, "plain")]:
        x, w = _randn(rows, k, seed=1).requires_grad_(), _randn(4, n, k, seed=2).requires_grad_()
        y = ops.grouped_mm(x, w, _ends(counts))
        dy = {"plain": lambda: _randn(rows, n, seed=3), "transposed": lambda: _randn(n, rows, seed=3).t(),
              "expanded": lambda: _randn(1, 1, seed=3).expand(rows, n)}[shape]()
        gx, gw = torch.autograd.grad(y, (x, w), dy)
        _close(gx, _dx(dy, w.detach(), counts), _dx(dy.abs(), w.detach().abs(), counts), n)
        _close(gw, _dw(dy, x.detach(), counts), _dw(dy.abs(), x.detach().abs(), counts), max(counts))
    only_w = torch.autograd.grad(ops.grouped_mm(x.detach(), w, _ends(counts)), w, dy)
    assert torch.equal(only_w[0], gw)


def test_gradients_against_differences():
    """<g, v> is the slope of the fp32 output's weighted sum along v: the function is linear in x and in w, so the
    difference over any step is exact but for the fp32 sums."""
    counts, n, k = [3, 20, 0, 9], 40, 56
    rows = sum(counts)
    ends = _ends(counts)
    # values on a coarse grid: x + v and w + v are exact in bf16
    grid = lambda *s, seed: (torch.randint(-8, 9, s, generator=torch.Generator().manual_seed(seed)) / 8).to(  # noqa: E731
        torch.bfloat16).to(DEV)
    x, vx, w, vw = grid(rows, k, seed=1), grid(rows, k, seed=2), grid(4, n, k, seed=3), grid(4, n, k, seed=4)
    dy = grid(rows, n, seed=5)
    f = lambda a, b: (ops.grouped_mm(a, b, ends, out_dtype=torch.float32).double() * dy.double()).sum()  # noqa: E731
    dx = ops.grouped_mm_dx(dy, w, ends, out_dtype=torch.float32).double()
    dw = ops.grouped_mm_dw(dy, x, ends, out_dtype=torch.float32).double()
    # products are multiples of 2^-6 (outputs) and 2^-9 (sums below), far inside 24 bits: every figure is exact
    assert (f(x + vx, w) - f(x, w) - (dx * vx.double()).sum()).abs().item() == 0
    assert (f(x, w + vw) - f(x, w) - (dw * vw.double()).sum()).abs().item() == 0


# ---------------------------------------------------------------- 8-bit integers
def _quant_ref(x):
    """The definition with IEEE fp32 steps, evaluated in 64 bits and rounded to 32 after each."""
    x = x.double().cpu()
    scale = torch.maximum(x.abs().amax(1) / 127, torch.tensor(1e-12, dtype=torch.float64)).float()
    q = (x / scale.double()[:, None]).float().double().round().clamp(-127, 127)
    return q.to(torch.int8), scale


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7168), (3, 7), (33, 129), (257, 64), (5, 1000), (64, 4096), (9, 8191),
                                       (3, 32768), (2, 70001), (5000, 64), (3001, 24), (1500, 2048), (700, 7168),
                                       (900, 16384)])
def test_quant_int8_is_exact(rows, cols, dtype):
    x = _randn(rows, cols, seed=rows + cols, dtype=dtype, std=3.0)
    if rows > 2:
        x[1] = 0
        x[2, cols // 2] = 3.0e4
    if cols > 200:                       # quotients on and next to a tie
        x[0, :201] = torch.arange(-100, 101).to(dtype).to(DEV) / 4
        x[0, 5] = 127 / 4
    q, s = ops.quant_int8(x)
    torch.cuda.synchronize()
    qr, sr = _quant_ref(x)
    assert torch.equal(s.cpu(), sr)
    assert torch.equal(q.cpu(), qr)


@pytest.mark.parametrize("steps", [0, 1, 3, 300])
def test_quant_int8_next_to_ties(steps):
    """Rows whose quotients lie on a tie or up to `steps` steps of x beside it, at scales of every size."""
    g = torch.Generator().manual_seed(steps)
    rows, cols = 600, 512
    top = torch.exp(torch.empty(rows, dtype=torch.float64).uniform_(-20, 60, generator=g)).float()
    scale = torch.maximum(top.double() / 127, torch.tensor(1e-12, dtype=torch.float64)).float()
    m = torch.randint(-127, 127, (rows, cols), generator=g)
    x = ((m + 0.5) * scale.double()[:, None]).float()
    x = (x.view(torch.int32) + torch.randint(-steps, steps + 1, (rows, cols), generator=g, dtype=torch.int32)).view(torch.float32)
    x[:, 7] = top
    q, s = ops.quant_int8(x.to(DEV))
    qr, sr = _quant_ref(x)
    assert torch.equal(s.cpu(), sr)
    assert torch.equal(q.cpu(), qr)


def test_quant_int8_strides_and_unaligned_rows():
    big = _randn(20, 700, seed=1)
    for at, cols in [(0, 256), (8, 513), (3, 100), (1, 699)]:
        x = big[:, at:at + cols]
        q = torch.full((20, cols + 5), 99, dtype=torch.int8, device=DEV)
        ops.quant_int8(x, q[:, 2:2 + cols])
        qr, _ = _quant_ref(x)
        assert torch.equal(q[:, 2:2 + cols].cpu(), qr)
        assert (q[:, :2] == 99).all() and (q[:, 2 + cols:] == 99).all()


def test_quant_int8_marks_rows_that_are_not_finite():
    x = _randn(6, 300, seed=1, dtype=torch.float32)
    x[1, 7], x[2, 0], x[3, 299] = float("nan"), float("inf"), float("-inf")
    x[4] = 1e-30
    q, s = ops.quant_int8(x)
    assert torch.isnan(s[1]) and torch.isinf(s[2]) and torch.isinf(s[3])
    assert s[4].item() == torch.tensor(1e-12).item() and not q[4].any()
    a = torch.zeros((6, 304), dtype=torch.int8, device=DEV)
    a[:, :300] = q
    w = torch.ones((16, 304), dtype=torch.int8, device=DEV)
    y = ops.int8_mm(a, s, w, torch.ones(16, device=DEV))
    assert torch.isnan(y[1:4]).all() and torch.isfinite(y[[0, 4, 5]]).all()


def _codes(*shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8).to(DEV)


def _scales(*shape, seed):
    return (torch.rand(shape, generator=torch.Generator().manual_seed(seed)) * 0.01 + 1e-4).to(DEV)


def _int8_ref(a, a_scale, w, w_scale, dtype):
    sums = (a.double() @ w.double().T).float()          # exact in 64 bits, one rounding
    return (sums * a_scale[:, None] * w_scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 4096, 512), (2, 129, 64), (17, 255, 1008), (33, 640, 2048),
                                   (300, 1001, 400), (1000, 384, 7168), (257, 128, 16), (1, 2048, 7168),
                                   (32, 130, 4096), (20, 1000, 2064), (1, 4096, 4096), (7, 64, 1024)])
def test_int8_mm_is_exact(m, n, k, dtype):
    a, w = _codes(m, k, seed=1), _codes(n, k, seed=2)
    sa, sw = _scales(m, seed=3), _scales(n, seed=4)
    y = ops.int8_mm(a, sa, w, sw, out_dtype=dtype)
    torch.cuda.synchronize()
    assert torch.equal(y, _int8_ref(a, sa, w, sw, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,pitch,offset", [(600, 201, 203, 1), (70, 1714, 1714, 0), (300, 66, 72, 0), (129, 65, 65, 3), (5, 33, 35, 1)])
def test_int8_outputs_that_start_anywhere(m, n, pitch, offset, dtype):
    a, a_scale, w, w_scale = _codes(m, 80, seed=1), _scales(m, seed=2), _codes(n, 80, seed=3), _scales(n, seed=4)
    flat = torch.full((offset + m * pitch + 8,), -7.0, device=DEV, dtype=dtype)
    out = flat.as_strided((m, n), (pitch, 1), offset)
    ops.int8_mm(a, a_scale, w, w_scale, out=out)
    assert torch.equal(out, _int8_ref(a, a_scale, w, w_scale, dtype))
    out.fill_(-7.0)
    assert (flat == -7.0).all()


def test_int8_sums_at_the_edge_of_32_bits():
    k = 131056
    a, w = torch.full((2, k), -128, dtype=torch.int8, device=DEV), torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    one = torch.ones(3, device=DEV)
    y = ops.int8_mm(a, one[:2], w, one, out_dtype=torch.float32)
    want = torch.tensor([128 * 128 * k, -128 * 127 * k, 128 * 128 * k], dtype=torch.float64).float()
    assert torch.equal(y.cpu(), want.expand(2, 3))


@pytest.mark.parametrize("counts,slack,n,k", [([1], 0, 16, 16), ([7, 0, 300, 17, 0, 1], 11, 201, 336),
                                              ([0, 0], 4, 64, 64), ([1] * 100 + [0] * 50, 3, 130, 256),
                                              ([700, 1, 64], 0, 512, 1040)])
def test_int8_grouped_mm_is_exact(counts, slack, n, k):
    rows = sum(counts) + slack
    a, w = _codes(rows, k, seed=1), _codes(len(counts), n, k, seed=2)
    sa, sw = _scales(rows, seed=3), _scales(len(counts), n, seed=4)
    y = ops.int8_grouped_mm(a, sa, w, sw, _ends(counts), out_dtype=torch.float32)
    for e, s in _spans(counts):
        assert torch.equal(y[s], _int8_ref(a[s], sa[s], w[e], sw[e], torch.float32)), e
    if slack:
        assert not y[-slack:].any()


def test_strided_integer_operands():
    wide_a, wide_w = _codes(40, 512, seed=1), _codes(3, 90, 640, seed=2)
    a, w = wide_a[:, 32:32 + 200], wide_w[:, 5:75, 16:216]
    sa, sw = _scales(40, seed=3), _scales(3, 70, seed=4)
    y = ops.int8_grouped_mm(a, sa, w, sw, _ends([11, 0, 29]), out_dtype=torch.float32)
    assert torch.equal(y[:11], _int8_ref(a[:11], sa[:11], w[0], sw[0], torch.float32))
    assert torch.equal(y[11:], _int8_ref(a[11:], sa[11:], w[2], sw[2], torch.float32))


# ---------------------------------------------------------------- used together
def _route(tokens, experts, top_k, seed):
    logits = _randn(tokens, experts, seed=seed, dtype=torch.float32)
    ids, wts = ops.route_topk(logits, top_k)
    order, expert_of, _ = ops.moe_align_block_size(ids, 1, experts)       # blocks of one row: sorted, no padding
    ends = torch.searchsorted(expert_of, torch.arange(experts, device=DEV, dtype=torch.int32), right=True)
    return ids, wts, order.long(), ends.to(torch.int32)


@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_a_routed_layer_and_its_gradients(tokens):
    """route -> sort -> gate/up product -> SiLU * up -> down product -> weighted sum, and its gradients, against the
    same layer with one dense product for each token and expert in 64 bits.

    The layer rounds h to bf16 and each product's output once, and the gradients pass the same roundings back: a chain
    of at most five roundings of relative size 2^-8, plus fp32 sums far below them.  Each enters a sum whose terms have
    independent signs, so the 2-norm of the difference stays below five times 2^-8 of the norm of the result."""
    cfg = configs.preset("tiny").shape
    e, h, inter, top_k = cfg.E, cfg.K, cfg.n_down, cfg.top_k
    ids, wts, order, ends = _route(tokens, e, top_k, seed=tokens)
    x = _randn(tokens, h, seed=1).requires_grad_()
    w1 = _randn(e, 2 * inter, h, seed=2, std=h ** -0.5).requires_grad_()
    w2 = _randn(e, h, inter, seed=3, std=inter ** -0.5).requires_grad_()

    gu = ops.grouped_mm(x[order // top_k], w1, ends)
    gate, up = gu.float().chunk(2, -1)
    y = ops.grouped_mm((torch.nn.functional.silu(gate) * up).to(torch.bfloat16), w2, ends)
    pairs = torch.empty_like(y).index_copy(0, order, y)
    out = (pairs.float().view(tokens, top_k, h) * wts[..., None]).sum(1)
    dout = _randn(tokens, h, seed=4, dtype=torch.float32)
    grads = torch.autograd.grad(out, (x, w1, w2), dout)

    xd, w1d, w2d = (t.detach().double().requires_grad_() for t in (x, w1, w2))
    want = 0
    for j in range(top_k):
        g2, u2 = torch.einsum("th,tnh->tn", xd, w1d[ids[:, j].long()]).chunk(2, -1)
        y2 = torch.einsum("ti,thi->th", torch.nn.functional.silu(g2) * u2, w2d[ids[:, j].long()])
        want = want + y2 * wts[:, j, None].double()
    want_grads = torch.autograd.grad(want, (xd, w1d, w2d), dout.double())
    for got, ref in zip((out, *grads), (want, *want_grads)):
        assert ((got.double() - ref).norm() / ref.norm()).item() < 5 * 2.0 ** -8


@pytest.mark.parametrize("tokens", [1, 130])
def test_a_routed_integer_layer(tokens):
    """The same layer with 8-bit weights and activations; the oracle takes the same codes and rounds where it does, so
    the layer's outputs differ from it by the fp32 SiLU's last bits, which can move a code by one: 1 / 127 of a row's
    largest value, in one of many terms."""
    cfg = configs.preset("tiny").shape
    e, h, inter, top_k = cfg.E, cfg.K, cfg.n_down, cfg.top_k
    ids, wts, order, ends = _route(tokens, e, top_k, seed=tokens + 50)
    x = _randn(tokens, h, seed=1)
    w1, s1 = ops.quant_int8(_randn(e * 2 * inter, h, seed=2))
    w2, s2 = ops.quant_int8(_randn(e * h, inter, seed=3))
    w1, s1, w2, s2 = w1.view(e, 2 * inter, h), s1.view(e, 2 * inter), w2.view(e, h, inter), s2.view(e, h)

    q, s = ops.quant_int8(x)
    rows = order // top_k
    gu = ops.int8_grouped_mm(q[rows], s[rows], w1, s1, ends, out_dtype=torch.float32)
    gate, up = gu.chunk(2, -1)
    hq, hs = ops.quant_int8(torch.nn.functional.silu(gate) * up)
    y = ops.int8_grouped_mm(hq, hs, w2, s2, ends)
    pairs = torch.empty_like(y).index_copy(0, order, y)
    out = ops.combine((pairs.view(tokens, top_k, h) * wts[..., None]).to(torch.bfloat16).view(-1, h), top_k)

    xd = q.double() * s.double()[:, None]
    want = torch.zeros((tokens, h), dtype=torch.float64, device=DEV)
    for j in range(top_k):
        g2, u2 = torch.einsum("th,tnh->tn", xd, (w1.double() * s1.double()[..., None])[ids[:, j].long()]).chunk(2, -1)
        h2 = torch.nn.functional.silu(g2) * u2
        hs2 = h2.abs().amax(1, keepdim=True) / 127
        h2 = (h2 / hs2).round() * hs2
        want += torch.einsum("ti,thi->th", h2, (w2.double() * s2.double()[..., None])[ids[:, j].long()]) * \
            wts[:, j, None].double()
    # bf16 roundings of y and of the weighted rows and of the sum: three times 2^-8
    assert ((out.double() - want).norm() / want.norm()).item() < 3 * 2.0 ** -8


# ---------------------------------------------------------------- streams, graphs
def test_other_stream_and_replayed_graph():
    counts = [40, 0, 3, 85]
    x, w, dy = _randn(128, 128, seed=1), _randn(4, 192, 128, seed=2), _randn(128, 192, seed=3)
    ends = _ends(counts)
    qa, sa = ops.quant_int8(x)
    qw, sw = ops.quant_int8(w.view(-1, 128))
    qw, sw = qw.view(4, 192, 128), sw.view(4, 192)
    run = lambda: (ops.grouped_mm(x, w, ends), ops.grouped_mm_dx(dy, w, ends), ops.grouped_mm_dw(dy, x, ends),  # noqa: E731
                   ops.int8_grouped_mm(qa, sa, qw, sw, ends), *ops.quant_int8(x))
    eager = run()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.synchronize()
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    # new routing, new rows: the captured calls read both from the device
    ends.copy_(_ends([1, 100, 0, 20]))
    x.copy_(_randn(128, 128, seed=11))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(held, run()):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    counts = [900, 0, 300, 700]
    x, w = _randn(1900, 512, seed=1), _randn(4, 768, 512, seed=2)
    ends = _ends(counts)
    want = ops.grouped_mm(x, w, ends)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.grouped_mm(x, w, ends))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_results_do_not_change_from_run_to_run():
    counts = [100, 0, 3, 85, 300]
    x, w, dy = _randn(488, 640, seed=1), _randn(5, 384, 640, seed=2), _randn(488, 384, seed=3)
    ends = _ends(counts)
    run = lambda: (ops.grouped_mm(x, w, ends), ops.grouped_mm_dx(dy, w, ends), ops.grouped_mm_dw(dy, x, ends))  # noqa: E731
    first = run()
    for _ in range(5):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)


def test_two_graphs_replayed_at_once():
    """Captured calls hold no workspace that another graph could share."""
    sets = []
    for seed, counts in ((1, [30, 0, 300, 70]), (2, [1, 1, 0, 6])):
        rows = sum(counts)
        sets.append((_randn(rows, 512, seed=seed), _randn(4, 640, 512, seed=seed + 10), _ends(counts),
                     _randn(rows, 640, seed=seed + 20)))
    run = lambda x, w, ends, dy: (ops.grouped_mm(x, w, ends), ops.grouped_mm_dx(dy, w, ends),  # noqa: E731
                                  ops.grouped_mm_dw(dy, x, ends), *ops.quant_int8(x))
    want = [run(*s) for s in sets]
    graphs, held, streams = [], [], [torch.cuda.Stream(DEV) for _ in sets]
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(run(*s))
    torch.cuda.synchronize()
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for h, w in zip(held, want):
        assert all(torch.equal(a, b) for a, b in zip(h, w))


def test_captured_training_step():
    """Forward and backward of leaves that no eager graph holds, captured and replayed with other values."""
    counts = [20, 0, 44]
    x, w, dy = _randn(64, 96, seed=1).requires_grad_(), _randn(3, 80, 96, seed=2).requires_grad_(), _randn(64, 80, seed=3)
    ends = _ends(counts)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.grouped_mm(x, w, ends), (x, w), dy)      # its graph is gone before the capture
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gx, gw = torch.autograd.grad(ops.grouped_mm(x, w, ends), (x, w), dy)
    with torch.no_grad():
        x.copy_(_randn(64, 96, seed=11))
        w.copy_(_randn(3, 80, 96, seed=12))
    graph.replay()
    torch.cuda.synchronize()
    xd, wd = x.detach(), w.detach()
    _close(gx, _dx(dy, wd, counts), _dx(dy.abs(), wd.abs(), counts), 80)
    _close(gw, _dw(dy, xd, counts), _dw(dy.abs(), xd.abs(), counts), 44)


def test_another_current_device(monkeypatch):
    """With another device current, the call switches to the tensors' one (here: told that another one is)."""
    x, w, ends = _randn(6, 64, seed=1), _randn(2, 48, 64, seed=2), _ends([4, 2])
    want = ops.grouped_mm(x, w, ends)
    switched = []
    device = torch.cuda.device
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", lambda i: switched.append(i) or device(i))
    got = ops.grouped_mm(x, w, ends)
    monkeypatch.undo()
    assert switched == [0] and torch.equal(got, want)


def test_refusals_of_the_wrappers():
    x, w, ends = _randn(8, 64, seed=1), _randn(2, 32, 64, seed=2), _ends([5, 3])
    dy = _randn(8, 32, seed=3)
    bad = [
        (lambda: ops.grouped_mm(x.float(), w, ends), "bf16 or fp16"),
        (lambda: ops.grouped_mm(x.half(), w, ends), "w must be"),
        (lambda: ops.grouped_mm(x, w[:, :, :32], ends), "summed axes"),
        (lambda: ops.grouped_mm(x[0], w, ends), "x must be"),
        (lambda: ops.grouped_mm(x.t(), w, ends), "x must be"),
        (lambda: ops.grouped_mm(x, w, ends.long()), "ends must be"),
        (lambda: ops.grouped_mm(x, w, ends[:1]), "ends must be"),
        (lambda: ops.grouped_mm(x, w, ends.cpu()), "ends must be"),
        (lambda: ops.grouped_mm(x, w, ends, out_dtype=torch.float16), "out_dtype"),
        (lambda: ops.grouped_mm(x, w, ends, out=torch.empty((8, 31), device=DEV, dtype=x.dtype)), "out must be"),
        (lambda: ops.grouped_mm(x, w, ends, out=x[:, :32]), "overlaps"),
        (lambda: ops.grouped_mm(x, w, ends, status=torch.zeros(1, device=DEV)), "status"),
        (lambda: ops.grouped_mm(x.requires_grad_(), w, ends, out=dy), "gradients"),
        (lambda: ops.grouped_mm_dx(dy, w.transpose(1, 2), ends), "w must be"),
        (lambda: ops.grouped_mm_dw(dy, x.detach()[:7], ends), "rows"),
        (lambda: ops.grouped_mm_dw(dy, x.detach().half(), ends), "x must be"),
        (lambda: ops.grouped_mm_dw(dy, x.detach(), ends[None]), "ends must be"),
        (lambda: ops.quant_int8(x.detach().double()), "2D"),
        (lambda: ops.quant_int8(x.detach().t()), "2D"),
        (lambda: ops.quant_int8(x.detach(), q=torch.empty((8, 63), dtype=torch.int8, device=DEV)), "bad q"),
        (lambda: ops.quant_int8(x.detach(), scale=torch.empty(7, device=DEV)), "scale must be"),
    ]
    a, s = ops.quant_int8(x.detach())
    wq, sw = ops.quant_int8(w.view(-1, 64))
    bad += [
        (lambda: ops.int8_mm(a, s, wq[:, :32], sw), "summed axes"),
        (lambda: ops.int8_mm(a, s[:7], wq, sw), "a_scale"),
        (lambda: ops.int8_mm(a, s, wq, sw[:5]), "w_scale"),
        (lambda: ops.int8_mm(a, s.double(), wq, sw), "a_scale"),
        (lambda: ops.int8_mm(a.float(), s, wq, sw), "a must be"),
        (lambda: ops.int8_mm(a, s, wq, sw, out_dtype=torch.int32), "out_dtype"),
        (lambda: ops.int8_grouped_mm(a, s, wq.view(2, 32, 64), sw, ends), "w_scale"),
        (lambda: ops.int8_grouped_mm(a, s, wq, sw.view(2, 32), ends), "w must be"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: ops.grouped_mm(x.detach().expand(8, 64)[:, 1:61], w[:, :, 1:61], ends),   # unaligned rows
                 lambda: ops.grouped_mm(_randn(1, 64).expand(8, 64), w, ends),                     # rows on one another
                 lambda: ops.grouped_mm(x.detach(), _randn(1, 32, 64).expand(2, 32, 64), ends),
                 lambda: ops.int8_mm(a[:, :24].contiguous(), s, wq[:, :24].contiguous(), sw)):
        with pytest.raises(Exception, match="16 bytes|16-byte"):
            call()


def test_quant_refuses_scales_on_its_operands():
    x = torch.zeros(8, 64, device=DEV)
    q = torch.zeros(8, 64, device=DEV, dtype=torch.int8)
    for scale in (x.view(-1)[:8], q.view(-1)[:32].view(torch.float32)):
        with pytest.raises(ValueError, match="scale overlaps"):
            ops.quant_int8(x, q=q, scale=scale)


def test_one_double_backward_is_refused():
    x, w = _randn(4, 64, seed=1).requires_grad_(), _randn(1, 32, 64, seed=2).requires_grad_()
    y = ops.grouped_mm(x, w, _ends([4]))
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), w)
