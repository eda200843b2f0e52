"""Calls of the expert-segment and integer products that are refused, through the C ABI: no device is touched."""
import pytest

from td_benchmark_b200 import _lib

BF16, FP16, FP32 = 0, 1, 2
P = 4096          # stands for an aligned address; every call below is refused before it is used

MM = dict(x=P, rows=8, ldx=64, w=P, experts=4, n=32, k=64, ldw=64, w_stride=2048, ends=P, in_type=BF16, out=P, ldo=64,
          out_type=BF16, clear=1, status=None, stream=None)
DW = dict(dy=P, lddy=32, x=P, ldx=64, rows=8, n=32, k=64, ends=P, experts=4, in_type=BF16, out=P, ldo=64,
          out_stride=2048, out_type=BF16, status=None, stream=None)
QUANT = dict(x=P, in_type=BF16, rows=4, cols=64, ldx=64, q=P, ldq=64, scale=P, status=None, stream=None)
INT8 = dict(a=P, a_scale=P, rows=8, lda=64, w=P, w_scale=P, experts=4, n=32, k=64, ldw=64, w_stride=2048, ends=P, out=P,
            ldo=32, out_type=BF16, clear=1, status=None, stream=None)


@pytest.fixture(autouse=True)
def _built():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libb2m.so not built")


def _refused(fn, base, change, match):
    with pytest.raises(_lib.B2MError, match=match) as e:
        _lib.call(fn, *dict(base, **change).values())
    assert e.value.code == 1          # an argument error, also where there is no GPU


COMMON = [
    (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(n=0), "extent|no rows"), (dict(k=0), "extent"),
    (dict(rows=-1), "extent"), (dict(rows=(1 << 30) + 1), "extent"), (dict(k=1 << 31, ldx=1 << 31, ldw=1 << 31), "extent"),
    (dict(ends=None), "ends"), (dict(out=None), "null output"), (dict(out=P + 1), "misaligned"),
    (dict(ldo=16), "output rows"), (dict(in_type=FP32), "neither"), (dict(in_type=7), "neither"),
    (dict(out_type=FP16), "output type"), (dict(out_type=9), "output type"),
]


@pytest.mark.parametrize("change,match", COMMON + [
    (dict(ldx=68), "rows of x"), (dict(ldx=56), "rows of x"), (dict(x=None), "x must not be null"),
    (dict(x=P + 8), "aligned"), (dict(w=P + 2), "aligned"), (dict(w=None), "w must not be null"),
    (dict(ldw=60), "rows of w"), (dict(w_stride=0), "experts of w"), (dict(w_stride=2049), "experts of w"),
    (dict(rows=1 << 30, n=1 << 20, ldo=1 << 20), "tiles")])
def test_grouped_mm_refuses(change, match):
    _refused("b2m_grouped_mm", MM, change, match)


@pytest.mark.parametrize("change,match", [(dict(ldx=24), "rows of dy"), (dict(x=None), "dy must not be null"),
                                          (dict(ends=None), "ends"), (dict(ldo=63), "output rows"),
                                          (dict(ldw=72 + 1), "rows of w")])
def test_grouped_mm_dx_refuses(change, match):
    _refused("b2m_grouped_mm_dx", dict(MM, ldx=32), change, match)


@pytest.mark.parametrize("change,match", [c for c in COMMON if "ldw" not in c[0]] + [
    (dict(lddy=36), "rows of dy"), (dict(ldx=68), "rows of x"), (dict(dy=P + 4), "dy must not be null"),
    (dict(out_stride=2047), "overlap"), (dict(ldo=48), "output rows")])
def test_grouped_mm_dw_refuses(change, match):
    _refused("b2m_grouped_mm_dw", DW, change, match)


@pytest.mark.parametrize("change,match", [(dict(cols=0), "bad shape"), (dict(rows=-1), "bad shape"),
                                          (dict(ldx=63), "bad shape"), (dict(ldq=63), "bad shape"),
                                          (dict(in_type=3), "input type"), (dict(x=None), "null"),
                                          (dict(q=None), "null"), (dict(scale=None), "null"),
                                          (dict(x=P + 1), "misaligned")])
def test_quant_i8_refuses(change, match):
    _refused("b2m_quant_i8", QUANT, change, match)


@pytest.mark.parametrize("change,match", [(dict(k=131072, lda=131072, ldw=131072), "32 bits"), (dict(lda=72), "rows of a"),
                                          (dict(ldw=65), "rows of w"), (dict(a_scale=None), "scales"),
                                          (dict(w_scale=None), "scales"), (dict(ends=None), "one expert"),
                                          (dict(out_type=3), "output type"), (dict(a=P + 8), "aligned"),
                                          (dict(w=P + 8), "aligned"), (dict(ldo=31), "output rows"),
                                          (dict(experts=0), "experts")])
def test_int8_mm_refuses(change, match):
    _refused("b2m_int8_mm", INT8, change, match)


def test_wrappers_refuse_host_tensors_and_wrong_shapes():
    import torch

    from td_benchmark_b200 import ops

    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((2, 32, 64), dtype=torch.bfloat16)
    ends = torch.tensor([2, 4], dtype=torch.int32)
    a, s = torch.zeros((4, 64), dtype=torch.int8), torch.zeros(4)
    for call in (lambda: ops.grouped_mm(x, w, ends), lambda: ops.grouped_mm_dx(x, w, ends),
                 lambda: ops.grouped_mm_dw(x, x, ends), lambda: ops.quant_int8(x), lambda: ops.int8_mm(a, s, a, s),
                 lambda: ops.int8_grouped_mm(a, s, a.view(2, 2, 64), s, ends)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("name", ["grouped_mm", "grouped_mm_dx", "grouped_mm_dw", "quant_int8", "int8_mm",
                                  "int8_grouped_mm"])
def test_every_wrapper_takes_a_status_word(name):
    """A wait that runs out is reported there and nowhere else."""
    import inspect

    from td_benchmark_b200 import ops

    assert inspect.signature(getattr(ops, name)).parameters["status"].default is None


def _bytes_of(t):
    import itertools

    at = {sum(i * s for i, s in zip(index, t.stride())) for index in itertools.product(*map(range, t.shape))}
    return {t.data_ptr() + i * t.element_size() + b for i in at for b in range(t.element_size())}


def test_tensors_that_share_no_byte():
    """Never called apart when they share one, and called apart when they are parts of one buffer's rows."""
    import random

    import torch

    from td_benchmark_b200 import ops

    buf = torch.zeros((6, 40), dtype=torch.bfloat16)
    cube = torch.zeros((3, 8, 20), dtype=torch.bfloat16)
    for a, b in [(buf[:, :16], buf[:, 16:]), (buf[:, 24:], buf[1:4, 8:24]), (buf[0], buf[2:]), (buf[:3], buf[3:]),
                 (cube[:, :4], cube[:, 4:]), (cube[..., :8], cube[..., 8:16]), (buf[:, :8], buf.view(torch.int8)[:, 64:]),
                 (buf[::2], buf[1::2]), (buf[:, :0], buf)]:
        assert ops._apart(a, b) and ops._apart(b, a) and not _bytes_of(a) & _bytes_of(b)
    for a, b in [(buf, buf), (buf[:, :17], buf[:, 16:]), (buf[:3], buf[2:]), (buf.view(-1)[:4], buf), (buf[0], buf[:1]),
                 (cube[0], cube[:, 4]), (buf[:1].expand(6, 40), buf[:, 39:])]:
        assert not ops._apart(a, b) and not ops._apart(b, a)
    rng = random.Random(1)
    flat, apart = torch.zeros(120, dtype=torch.int16), 0
    for _ in range(3000):
        views = []
        for _ in range(2):
            shape = [rng.randrange(1, 4) for _ in range(rng.randrange(1, 4))]
            strides = [rng.choice([0, 1, 2, 5, 8, 10, 16, 20]) for _ in shape[1:]] + [1]
            room = 119 - sum((n - 1) * s for n, s in zip(shape, strides))
            views.append(flat.as_strided(shape, strides, rng.randrange(0, room)))
        if ops._apart(*views):
            apart += 1
            assert not _bytes_of(views[0]) & _bytes_of(views[1]), views
    assert apart > 500


@pytest.mark.parametrize("fn,base,names", [("b2m_grouped_mm", MM, ("ends", "status")),
                                           ("b2m_grouped_mm_dx", dict(MM, ldx=32), ("ends", "status")),
                                           ("b2m_grouped_mm_dw", DW, ("ends", "status")),
                                           ("b2m_quant_i8", QUANT, ("scale", "status")),
                                           ("b2m_int8_mm", INT8, ("ends", "a_scale", "w_scale", "status"))])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_words_that_start_anywhere_are_refused(fn, base, names, off):
    """A 32-bit access at such an address would fault."""
    for name in names:
        _refused(fn, base, {name: P + off}, "4-byte aligned")


@pytest.mark.parametrize("far", [(1 << 38) + 8, 1 << 59, 1 << 61, (1 << 62) - 16, 1 << 62, (1 << 63) - 16])
def test_strides_whose_products_pass_64_bits_are_refused(far):
    """Offsets are row times stride in 64 bits: a stride that no memory holds must not wrap into one that looks right."""
    for fn, base, names in [("b2m_grouped_mm", MM, ("ldx", "ldw", "w_stride", "ldo")),
                            ("b2m_grouped_mm_dx", dict(MM, ldx=32), ("ldx", "ldw", "w_stride", "ldo")),
                            ("b2m_grouped_mm_dw", DW, ("lddy", "ldx", "ldo", "out_stride")),
                            ("b2m_quant_i8", QUANT, ("ldx", "ldq")), ("b2m_int8_mm", INT8, ("lda", "ldw", "w_stride", "ldo"))]:
        for name in names:
            _refused(fn, base, {name: far}, "apart|bad shape")
    _refused("b2m_grouped_mm_dw", DW, dict(n=5, ldo=1 << 62, lddy=32), "apart")


@pytest.mark.parametrize("change", [dict(out_stride=32, ldo=128), dict(out_stride=64, ldo=255), dict(out_stride=63, ldo=4096),
                                    dict(out_stride=2047, ldo=64)])
def test_weight_gradients_whose_experts_overlap_are_refused(change):
    """Neither one behind the other nor row by row between the others."""
    _refused("b2m_grouped_mm_dw", DW, change, "overlap")
