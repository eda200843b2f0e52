"""torch-tensor wrappers over the b2m C ABI.

Each wrapper checks shapes/dtypes/devices, then enqueues the kernel on the
current CUDA stream of the tensors' device.  Outputs may be passed in (the layer
pre-allocates everything once); when omitted they are allocated here.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib

FP8 = torch.float8_e4m3fn
BLOCK = 128

STATUS_NAMES = {
    0x101: "TIMEOUT_PRODUCER", 0x102: "TIMEOUT_MMA", 0x103: "TIMEOUT_EPILOGUE", 0x104: "TIMEOUT_PEER",
    0x105: "TIMEOUT_DRAIN", 0x201: "BAD_ROUTING",
}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _cuda(t: torch.Tensor, name: str) -> None:
    _need(t.is_cuda, f"{name} must be a CUDA tensor")


def new_status(device) -> torch.Tensor:
    return torch.zeros(1, dtype=torch.int32, device=device)


def check_status(status: torch.Tensor, what: str = "b2m kernel") -> None:
    """Synchronise on the status word and raise if a kernel recorded an error."""
    code = int(status.item())
    if code:
        status.zero_()
        raise RuntimeError(f"{what}: device status 0x{code:x} ({STATUS_NAMES.get(code, 'unknown')})")


def quant_g128(x: torch.Tensor, q: torch.Tensor | None = None, scale: torch.Tensor | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [rows, cols] -> (e4m3 [rows, cols], fp32 [rows, ceil(cols/128)])."""
    _cuda(x, "x")
    _need(x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1, "x must be 2D bf16 with unit column stride")
    rows, cols = x.shape
    groups = (cols + BLOCK - 1) // BLOCK
    if q is None:
        q = torch.empty((rows, cols), dtype=FP8, device=x.device)
    if scale is None:
        scale = torch.empty((rows, groups), dtype=torch.float32, device=x.device)
    _need(q.shape == (rows, cols) and q.stride(1) == 1 and q.element_size() == 1, "bad q buffer")
    _need(scale.shape[0] == rows and scale.shape[1] >= groups and scale.stride(1) == 1 and
          scale.dtype == torch.float32, "bad scale buffer")
    _lib.call("b2m_quant_g128", x.data_ptr(), rows, cols, x.stride(0), q.data_ptr(), q.stride(0),
              scale.data_ptr(), scale.stride(0), _stream(x.device))
    return q, scale


def quant_g128_t(x: torch.Tensor, q: torch.Tensor, scale_t: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [rows, cols] -> e4m3 q [rows, cols] and K-block-major fp32 scale_t [cols/128, >= rows]."""
    _cuda(x, "x")
    _need(x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1, "x must be 2D bf16 with unit column stride")
    rows, cols = x.shape
    _need(scale_t.shape[0] == (cols + BLOCK - 1) // BLOCK and scale_t.shape[1] >= rows and scale_t.stride(1) == 1,
          "scale_t must be [cols/128, >= rows]")
    _lib.call("b2m_quant_g128_t", x.data_ptr(), rows, cols, x.stride(0), q.data_ptr(), q.stride(0),
              scale_t.data_ptr(), scale_t.stride(0), _stream(x.device))
    return q, scale_t


def quant_dispatch(x: torch.Tensor, pair_pos: torch.Tensor, top_k: int, a_sorted: torch.Tensor,
                   a_scale_t: torch.Tensor, q_tok: torch.Tensor | None = None,
                   scale_tok_t: torch.Tensor | None = None) -> None:
    """Quantise bf16 tokens and write codes/scales to the sorted rows of their pairs (+ optional token order)."""
    _cuda(x, "x")
    tokens, hidden = x.shape
    rows_cap = a_sorted.shape[0]
    _need(x.dtype == torch.bfloat16 and x.stride(1) == 1, "x must be bf16 with unit column stride")
    _need(pair_pos.dtype == torch.int32 and pair_pos.numel() == tokens * top_k, "pair_pos must be int32 [T*k]")
    _need(a_sorted.shape[1] == hidden and tuple(a_scale_t.shape) == (hidden // BLOCK, rows_cap),
          "a_sorted [rows_cap, H] / a_scale_t [H/128, rows_cap] mismatch")
    ld_tok = 0
    if q_tok is not None:
        _need(q_tok.shape[1] == hidden and q_tok.shape[0] >= tokens and scale_tok_t.shape[1] >= tokens,
              "bad token-order outputs")
        ld_tok = scale_tok_t.stride(0)
    _lib.call("b2m_quant_dispatch", x.data_ptr(), tokens, hidden, x.stride(0), pair_pos.data_ptr(), top_k,
              a_sorted.data_ptr(), a_scale_t.data_ptr(), rows_cap, _ptr(q_tok), _ptr(scale_tok_t), ld_tok,
              _stream(x.device))


def dispatch_rows(xq: torch.Tensor, xs: torch.Tensor, pair_pos: torch.Tensor, top_k: int, a_sorted: torch.Tensor,
                  a_scale_t: torch.Tensor) -> None:
    """Quantised token rows (+ row-major scales) -> sorted rows of their pairs."""
    _cuda(xq, "xq")
    tokens, hidden = xq.shape
    rows_cap = a_sorted.shape[0]
    _need(xq.is_contiguous() and xs.is_contiguous() and tuple(xs.shape) == (tokens, hidden // BLOCK),
          "xq / xs must be contiguous [T, H] / [T, H/128]")
    _need(pair_pos.dtype == torch.int32 and pair_pos.numel() == tokens * top_k, "pair_pos must be int32 [T*k]")
    _lib.call("b2m_dispatch_rows", xq.data_ptr(), xs.data_ptr(), tokens, hidden, pair_pos.data_ptr(), top_k,
              a_sorted.data_ptr(), a_scale_t.data_ptr(), rows_cap, _stream(xq.device))


def align_sizes(numel: int, num_experts: int, block_size: int) -> tuple[int, int]:
    """Buffer sizes of moe_align_block_size (vLLM moe_align_block_size.py:74-88)."""
    max_padded = numel + num_experts * (block_size - 1)
    if numel < num_experts:
        max_padded = min(numel * block_size, max_padded)
    return max_padded, (max_padded + block_size - 1) // block_size


def moe_align_block_size(topk_ids: torch.Tensor, block_size: int, num_experts: int,
                         expert_map: torch.Tensor | None = None,
                         out: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                         pair_pos: torch.Tensor | None = None, block_pairs: torch.Tensor | None = None
                         ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Same signature and outputs as vLLM's ``moe_align_block_size`` (without the padding flags).

    ``pair_pos`` (int32 [numel], optional) also receives each pair's sorted position (-1: non-local);
    ``block_pairs`` (int32 [1 + 2*nblk], optional) the block-pair work list of the paired-CTA GEMMs."""
    _cuda(topk_ids, "topk_ids")
    _need(topk_ids.dtype == torch.int32 and topk_ids.is_contiguous(), "topk_ids must be contiguous int32")
    numel = topk_ids.numel()
    cap, nblk = align_sizes(numel, num_experts, block_size)
    if out is None:
        sorted_ids = torch.empty(cap, dtype=torch.int32, device=topk_ids.device)
        expert_ids = torch.empty(nblk, dtype=torch.int32, device=topk_ids.device)
        ntpp = torch.empty(1, dtype=torch.int32, device=topk_ids.device)
    else:
        sorted_ids, expert_ids, ntpp = out
    if expert_map is not None:
        _need(expert_map.dtype == torch.int32 and expert_map.numel() >= num_experts, "expert_map must be int32 [E]")
    if pair_pos is not None:
        _need(pair_pos.dtype == torch.int32 and pair_pos.numel() == numel, "pair_pos must be int32 [numel]")
    if block_pairs is not None:
        _need(block_pairs.dtype == torch.int32 and block_pairs.numel() >= 1 + 2 * expert_ids.numel(),
              "block_pairs must be int32 [1 + 2*len(expert_ids)]")
    _lib.call("b2m_align", topk_ids.data_ptr(), numel, num_experts, block_size, _ptr(expert_map),
              sorted_ids.data_ptr(), sorted_ids.numel(), expert_ids.data_ptr(), expert_ids.numel(),
              ntpp.data_ptr(), _ptr(pair_pos), _ptr(block_pairs), _stream(topk_ids.device))
    return sorted_ids, expert_ids, ntpp


def w1_interleave(w1: torch.Tensor, w1_scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[E, 2I, H] gate-then-up -> 128-row interleaved gate/up layout (+ scales)."""
    _cuda(w1, "w1")
    e, n2, h = w1.shape
    _need(n2 % 256 == 0 and h % 128 == 0 and w1.is_contiguous() and w1_scale.is_contiguous(),
          "w1 must be contiguous [E, 2I, H] with I % 128 == 0 and H % 128 == 0")
    _need(tuple(w1_scale.shape) == (e, n2 // 128, h // 128), "w1_scale must be [E, 2I/128, H/128]")
    out = torch.empty_like(w1)
    out_s = torch.empty_like(w1_scale)
    _lib.call("b2m_w1_interleave", w1.data_ptr(), w1_scale.data_ptr(), e, n2 // 2, h, out.data_ptr(),
              out_s.data_ptr(), _stream(w1.device))
    return out, out_s


def gemm1(a_sorted: torch.Tensor, a_scale_t: torch.Tensor, w1i: torch.Tensor, w1i_scale: torch.Tensor,
          expert_ids: torch.Tensor, ntpp: torch.Tensor, out_q: torch.Tensor | None = None,
          out_scale_t: torch.Tensor | None = None, status: torch.Tensor | None = None,
          block_pairs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Gate/up grouped GEMM + SiLU*mul + 1x128 requant on expert-sorted A.

    a_sorted e4m3 [rows_cap, H], a_scale_t fp32 [H/128, rows_cap] -> (q [rows_cap, I], scale_t [I/128, rows_cap])."""
    _cuda(a_sorted, "a_sorted")
    rows_cap, hidden = a_sorted.shape
    e, n2, h2 = w1i.shape
    inter = n2 // 2
    _need(h2 == hidden and a_sorted.is_contiguous() and w1i.is_contiguous(), "A / W1 shape mismatch")
    _need(a_scale_t.is_contiguous() and tuple(a_scale_t.shape) == (hidden // 128, rows_cap),
          "a_scale_t must be [H/128, rows_cap]")
    _need(expert_ids.numel() * 128 >= rows_cap, "expert_ids shorter than rows_cap/128")
    if out_q is None:
        out_q = torch.empty((rows_cap, inter), dtype=FP8, device=a_sorted.device)
    if out_scale_t is None:
        out_scale_t = torch.empty((inter // 128, rows_cap), dtype=torch.float32, device=a_sorted.device)
    _lib.call("b2m_gemm1", a_sorted.data_ptr(), a_scale_t.data_ptr(), rows_cap, hidden, w1i.data_ptr(),
              w1i_scale.data_ptr(), e, inter, expert_ids.data_ptr(), ntpp.data_ptr(), _ptr(block_pairs),
              out_q.data_ptr(), out_scale_t.data_ptr(), _ptr(status), _stream(a_sorted.device))
    return out_q, out_scale_t


def gemm2(a_q: torch.Tensor, a_scale_t: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
          sorted_ids: torch.Tensor, expert_ids: torch.Tensor, ntpp: torch.Tensor, numel: int,
          topk_weights: torch.Tensor | None, out: torch.Tensor | None = None,
          status: torch.Tensor | None = None, block_pairs: torch.Tensor | None = None,
          cols: tuple[int, int] | None = None, max_ctas: int = 0) -> torch.Tensor:
    """Down grouped GEMM, routed weight in the epilogue.  Returns bf16 [numel, H] indexed by flat pair."""
    _cuda(a_q, "a_q")
    rows_cap, inter = a_q.shape
    e, hidden, i2 = w2.shape
    _need(i2 == inter and w2.is_contiguous() and a_q.is_contiguous(), "A / W2 shape mismatch")
    _need(tuple(a_scale_t.shape) == (inter // 128, rows_cap), "a_scale_t must be [I/128, rows_cap]")
    if topk_weights is not None:
        _need(topk_weights.dtype == torch.float32 and topk_weights.is_contiguous() and
              topk_weights.numel() == numel, "topk_weights must be contiguous fp32 with numel entries")
    if out is None:
        out = torch.empty((numel, hidden), dtype=torch.bfloat16, device=a_q.device)
    _lib.call("b2m_gemm2", a_q.data_ptr(), a_scale_t.data_ptr(), rows_cap, inter, w2.data_ptr(), w2_scale.data_ptr(),
              e, hidden, sorted_ids.data_ptr(), expert_ids.data_ptr(), ntpp.data_ptr(), _ptr(block_pairs), numel,
              _ptr(topk_weights), out.data_ptr(), 0 if cols is None else cols[0], 0 if cols is None else cols[1],
              max_ctas, _ptr(status), _stream(a_q.device))
    return out


def combine(staged: torch.Tensor, top_k: int, topk_ids: torch.Tensor | None = None,
            expert_map: torch.Tensor | None = None, shared: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [T*k, H] -> bf16 [T, H]: fp32 sum over the k slots (+ shared), one rounding."""
    _cuda(staged, "staged")
    pairs, hidden = staged.shape
    tokens = pairs // top_k
    if out is None:
        out = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=staged.device)
    _need(out.shape[0] >= tokens and out.stride(1) == 1, "bad combine output")
    _lib.call("b2m_combine", staged.data_ptr(), tokens, top_k, hidden, _ptr(topk_ids), _ptr(expert_map),
              _ptr(shared), out.data_ptr(), out.stride(0), _stream(staged.device))
    return out


def route_topk(logits: torch.Tensor, top_k: int, bias: torch.Tensor | None = None,
               out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 router logits [T, E] (+ per-expert bias [E]) -> (int32 ids [T, k], fp32 weights [T, k]):
    softmax, top-k in descending order, renormalised (``moe_bench/data/routing.py:58-64``)."""
    _cuda(logits, "logits")
    _need(logits.dtype == torch.float32 and logits.dim() == 2 and logits.is_contiguous(),
          "logits must be contiguous fp32 [T, E]")
    tokens, experts = logits.shape
    if bias is not None:
        _need(bias.dtype == torch.float32 and bias.numel() == experts and bias.is_contiguous(), "bias must be fp32 [E]")
    if out is None:
        ids = torch.empty((tokens, top_k), dtype=torch.int32, device=logits.device)
        wts = torch.empty((tokens, top_k), dtype=torch.float32, device=logits.device)
    else:
        ids, wts = out
        _need(ids.dtype == torch.int32 and wts.dtype == torch.float32 and ids.is_contiguous() and wts.is_contiguous()
              and tuple(ids.shape) == (tokens, top_k) and tuple(wts.shape) == (tokens, top_k),
              "out must be contiguous int32 / fp32 [T, k]")
    _lib.call("b2m_route_topk", logits.data_ptr(), tokens, experts, top_k, _ptr(bias), ids.data_ptr(), wts.data_ptr(),
              _stream(logits.device))
    return ids, wts


# ---------------------------------------------------------------- products over expert segments, 8-bit integers
# One-token calls take a few microseconds on the GPU, so these wrappers keep the host's part short: messages are made
# only when a check fails, and the device is switched only when it is not the current one.
TYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
FLOATS = (torch.bfloat16, torch.float16, torch.float32)


_tracing, _dispatch_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack


# Callers come here only when an input requires gradients, an output is given or a forward-mode level is open: the call
# itself would take 0.3 us of each of theirs.
def _no_gradient(what: str, *tensors: torch.Tensor | None) -> None:
    """Refuse tensors whose gradient the call would drop: it returns, or writes, values that no graph leads to."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what} is not differentiable: call it with detached tensors or under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _no_tangent(what, *tensors)


def _no_tangent(what: str, *tensors: torch.Tensor | None) -> None:
    """The same for forward-mode derivatives, whose tensors do not say that they require gradients."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} has no forward-mode derivative")


def _recording() -> bool:
    """Whether torch.fx records the operations of real tensors (of tensors without memory, data_ptr raises)."""
    return torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None


def _launch(device: torch.device, name: str, *args) -> None:
    """The C call on the tensors' device and its current stream."""
    if _tracing() or (_dispatch_modes() and _recording()):
        raise RuntimeError(f"{name}: a trace would keep the output's allocation and lose the kernel")
    index = device.index
    if index == torch._C._cuda_getDevice():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
        return
    with torch.cuda.device(index):
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _row_stride(stride: int, rows: int, cols: int, size: int) -> int:
    """Stride of an axis with ``rows`` entries; of one entry (whose stride says nothing) the smallest that the kernels
    take for rows of ``cols`` elements of ``size`` bytes."""
    return stride if rows > 1 else (cols * size + 15) // 16 * 16 // size


def _ldo(out: torch.Tensor) -> int:
    """Elements between an output's rows."""
    return out.stride(-2) if out.shape[-2] > 1 else out.shape[-1]


def _operand(t: torch.Tensor, name: str, dim: int, dtype: torch.dtype, device: torch.device) -> tuple:
    """Strides of a checked operand."""
    strides = t.stride()
    if len(strides) != dim or t.dtype is not dtype or t.device != device or (strides[-1] != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name} must be {dim}-D {dtype} on {device} with unit stride along its last axis")
    return strides


def _vector(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype, device: torch.device) -> None:
    if t.dtype is not dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} {list(shape)} on {device}")


def _status_word(status: torch.Tensor, device: torch.device) -> int:
    _need(status.dtype == torch.int32 and status.device == device and status.numel() >= 1,
          f"status must be int32 [1] on {device}")
    return status.data_ptr()


def _extent(t: torch.Tensor) -> tuple[int, int]:
    """First byte and the byte behind the last one that a tensor reaches."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share no byte: one lies behind the other, or they are parts of rows (or of other runs) that
    repeat at the same distance, as the halves of one buffer's columns are."""
    (lo, hi), (start, stop) = _extent(a), _extent(b)
    if hi <= start or stop <= lo:
        return True
    axes = [[(n, s * t.element_size()) for n, s in zip(t.shape, t.stride()) if n > 1 and s > 0] for t in (a, b)]
    for pitch in {s for of in axes for _, s in of}:
        first, second = (t.element_size() + sum((n - 1) * s for n, s in of if s % pitch) for t, of in zip((a, b), axes))
        at = (start - lo) % pitch                    # b's run behind a's, within a pitch
        if first <= at and at + second <= pitch:
            return True
    return False


def _output(out: torch.Tensor | None, shape: tuple, dtypes: tuple, out_dtype: torch.dtype | None,
            device: torch.device, inputs: tuple) -> torch.Tensor:
    """``out`` checked, or a new tensor.  inputs: the tensors that it must not overlap, the first one on its device."""
    if out is None:
        dtype = dtypes[0] if out_dtype is None else out_dtype
        if dtype not in dtypes:
            raise ValueError(f"out_dtype must be one of {list(dtypes)}")
        return inputs[0].new_empty(shape, dtype=dtype)
    _need(out_dtype is None or out_dtype == out.dtype, "out_dtype differs from out's")
    _need(tuple(out.shape) == shape and out.dtype in dtypes and out.device == device and
          (shape[-1] <= 1 or out.stride(-1) == 1),
          f"out must be {list(shape)} of {list(dtypes)} on {device} with unit stride along its last axis")
    for t in inputs:
        _need(_apart(out, t), "out overlaps an input")
    increment_version(out)          # a graph that saved its old values must not use the new ones
    return out


def _rows_times_weights(entry: str, name: str, x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor, summed: int,
                        out: torch.Tensor | None, out_dtype: torch.dtype | None, status: torch.Tensor | None
                        ) -> torch.Tensor:
    """x [T, .] times w [E, N, K] of its segment, summed over axis ``summed`` of w."""
    dtype, device = x.dtype, x.device
    if not x.is_cuda or (dtype is not torch.bfloat16 and dtype is not torch.float16):
        raise ValueError(f"{name} must be a CUDA tensor, bf16 or fp16")
    ldx, _ = _operand(x, name, 2, dtype, device)
    w_stride, ldw, _ = _operand(w, "w", 3, dtype, device)
    experts, n, k = w.shape
    rows, width = x.shape
    if width != (k if summed == 2 else n):
        raise ValueError(f"{name} is {list(x.shape)} and w {list(w.shape)}: the summed axes differ")
    _vector(ends, "ends", (experts,), torch.int32, device)
    cols = n if summed == 2 else k
    if out is None and (out_dtype is None or out_dtype is dtype):
        y = torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)   # 0.3 us less than new_empty
        ldo, code = cols, TYPE_CODES[dtype]
    else:
        y = _output(out, (rows, cols), (dtype, torch.float32), out_dtype, device, (x, w, ends))
        ldo, code = _ldo(y), TYPE_CODES[y.dtype]
    ldw = _row_stride(ldw, n, k, 2)
    _launch(device, entry, x.data_ptr(), rows, _row_stride(ldx, rows, width, 2), w.data_ptr(), experts, n, k, ldw,
            w_stride if experts > 1 else n * ldw, ends.data_ptr(), TYPE_CODES[dtype], y.data_ptr(), ldo, code,
            out is None, None if status is None else _status_word(status, device))
    return y


def grouped_mm(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor, out: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Rows sorted by expert times that expert's weights: ``y[t] = x[t] @ w[e].T`` for rows ``ends[e-1] <= t < ends[e]``.

    x bf16 / fp16 [T, K], w the same type [E, N, K], ends int32 [E] on the device (cumulative row counts; empty
    segments allowed, E <= 1024) -> [T, N] of the input type or fp32.  No segment is padded and nothing is read back
    to the host.  Rows behind ``ends[-1]`` are zero in an output allocated here and left alone in ``out``, which may
    lie beside an input in one buffer (columns next to its columns) but not on it.  Rows of x and w are a multiple of
    16 bytes apart and 16-byte aligned.  ``status`` (``new_status``) records ends that are out of order, which are
    otherwise taken as the nearest ones in order, and waits that ran out of their limit and left the output
    unfinished; a backward pass records both in the same word.

    Differentiable (in reverse mode, once) in x and w without ``out`` and ``out_dtype``; a weight gradient covers every
    expert (zero where a segment is empty).  As with any autograd function, a backward pass is captured into a CUDA
    graph only when no graph of the same leaves that was recorded outside the capture is still alive."""
    if forward_ad._current_level >= 0:
        _no_tangent("grouped_mm", x, w)
    if (x.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        _need(out is None and out_dtype in (None, x.dtype), "gradients need out=None and the input's type as out_dtype")
        return _GroupedMM.apply(x, w, ends, status)
    if out is not None:
        _no_gradient("grouped_mm into out", out)
    return _rows_times_weights("b2m_grouped_mm", "x", x, w, ends, 2, out, out_dtype, status)


def grouped_mm_dx(dy: torch.Tensor, w: torch.Tensor, ends: torch.Tensor, out: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``grouped_mm``'s rows: ``dx[t] = dy[t] @ w[e]``.  dy [T, N], w [E, N, K] -> [T, K]; types, strides,
    ends, status and the rows behind ``ends[-1]`` as there.  Not differentiable itself: tensors that require gradients
    are refused."""
    if dy.requires_grad or w.requires_grad or out is not None or forward_ad._current_level >= 0:
        _no_gradient("grouped_mm_dx", dy, w, out)
    return _rows_times_weights("b2m_grouped_mm_dx", "dy", dy, w, ends, 1, out, out_dtype, status)


def grouped_mm_dw(dy: torch.Tensor, x: torch.Tensor, ends: torch.Tensor, out: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``grouped_mm``'s weights: ``dw[e] = dy[seg e].T @ x[seg e]``, zero for an empty segment.

    dy [T, N], x [T, K] -> [E, N, K] of the input type or fp32; types, strides, ends and status as there.  Rows behind
    ``ends[-1]`` enter no sum, whatever they hold.  Not differentiable itself: tensors that require gradients are
    refused."""
    if dy.requires_grad or x.requires_grad or out is not None or forward_ad._current_level >= 0:
        _no_gradient("grouped_mm_dw", dy, x, out)
    dtype, device = dy.dtype, dy.device
    if not dy.is_cuda or (dtype is not torch.bfloat16 and dtype is not torch.float16):
        raise ValueError("dy must be a CUDA tensor, bf16 or fp16")
    lddy, _ = _operand(dy, "dy", 2, dtype, device)
    ldx, _ = _operand(x, "x", 2, dtype, device)
    rows, n = dy.shape
    k = x.shape[1]
    if x.shape[0] != rows:
        raise ValueError(f"dy has {rows} rows and x {x.shape[0]}")
    _need(ends.dim() == 1, "ends must be int32 [E]")
    experts = ends.shape[0]
    _vector(ends, "ends", (experts,), torch.int32, device)
    if out is None and (out_dtype is None or out_dtype is dtype):
        out, ldo, stride = torch.empty_strided((experts, n, k), (n * k, k, 1), dtype=dtype, device=device), k, n * k
    else:
        out = _output(out, (experts, n, k), (dtype, torch.float32), out_dtype, device, (dy, x, ends))
        ldo = _ldo(out)
        stride = out.stride(0) if experts > 1 else n * ldo
    _launch(device, "b2m_grouped_mm_dw", dy.data_ptr(), _row_stride(lddy, rows, n, 2), x.data_ptr(),
            _row_stride(ldx, rows, k, 2), rows, n, k, ends.data_ptr(), experts, TYPE_CODES[dtype], out.data_ptr(), ldo,
            stride, TYPE_CODES[out.dtype],
            None if status is None else _status_word(status, device))
    return out


def _kernel_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself when the kernels can read its rows, else a copy whose rows are (a gradient that torch hands over
    may be expanded, transposed or of a width that is no multiple of 16 bytes; saved tensors come back in another layout
    when hooks kept them elsewhere)."""
    shape, strides = t.shape, t.stride()
    rows, cols = shape[-2], shape[-1]
    if (strides[-1] == 1 or cols <= 1) and (rows <= 1 or (strides[-2] >= cols and strides[-2] % 8 == 0)) and \
            (len(shape) == 2 or shape[0] <= 1 or (strides[0] > 0 and strides[0] % 8 == 0)) and t.data_ptr() % 16 == 0:
        return t
    return torch.empty((*shape[:-1], (cols + 7) // 8 * 8), dtype=t.dtype, device=t.device)[..., :cols].copy_(t)


class _GroupedMM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, ends, status):
        y = grouped_mm(x.detach(), w.detach(), ends, status=status)
        ctx.save_for_backward(x, w, ends)
        ctx.status = status          # not among the saved tensors: the kernels may write to it
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, ends = ctx.saved_tensors
        x, w, dy = _kernel_rows(x), _kernel_rows(w), _kernel_rows(dy)
        dx = grouped_mm_dx(dy, w, ends, status=ctx.status) if ctx.needs_input_grad[0] else None
        dw = grouped_mm_dw(dy, x, ends, status=ctx.status) if ctx.needs_input_grad[1] else None
        return dx, dw, None, None


def quant_int8(x: torch.Tensor, q: torch.Tensor | None = None, scale: torch.Tensor | None = None,
               status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 / fp16 / fp32 [rows, cols] -> (int8 [rows, cols], fp32 [rows]): ``scale = max(amax / 127, 1e-12)``,
    ``q = rne(x / scale)`` within +-127, both divisions IEEE fp32.

    Token codes of activations, or channel codes of weights (one row for each output channel).  A row that holds a
    NaN (an infinity) gets a NaN (infinite) scale, and a product with it becomes NaN.  Not differentiable: an x that
    requires gradients is refused."""
    if x.requires_grad or scale is not None or forward_ad._current_level >= 0:
        _no_gradient("quant_int8", x, scale)
    code, device = TYPE_CODES.get(x.dtype), x.device
    strides = x.stride()
    if not x.is_cuda or code is None or len(strides) != 2 or (strides[1] != 1 and x.shape[1] > 1):
        raise ValueError("x must be a CUDA tensor, 2D bf16, fp16 or fp32 with unit column stride")
    rows, cols = x.shape
    if q is None:
        q = torch.empty_strided((rows, cols), (cols, 1), dtype=torch.int8, device=device)
        ldq = cols
    else:
        ldq, _ = _operand(q, "q", 2, torch.int8, device)
        ldq = ldq if rows > 1 else cols
        _need(tuple(q.shape) == (rows, cols) and ldq >= cols, "bad q buffer")
        _need(_apart(q, x), "q overlaps x")
        increment_version(q)
    if scale is None:
        scale = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=device)
    else:
        _vector(scale, "scale", (rows,), torch.float32, device)
        _need(_apart(scale, x) and _apart(scale, q), "scale overlaps x or q")
        increment_version(scale)
    _launch(device, "b2m_quant_i8", x.data_ptr(), code, rows, cols, strides[0] if rows > 1 else cols, q.data_ptr(), ldq,
            scale.data_ptr(), None if status is None else _status_word(status, device))
    return q, scale


def _int8(a, a_scale, w, w_scale, experts, n, k, w_stride, ldw, ends, out, out_dtype, status):
    if a_scale.requires_grad or w_scale.requires_grad or out is not None or forward_ad._current_level >= 0:
        _no_gradient("int8_mm" if ends is None else "int8_grouped_mm", a_scale, w_scale, out)
    device = a.device
    lda, _ = _operand(a, "a", 2, torch.int8, device)
    rows, width = a.shape
    if width != k:
        raise ValueError(f"a is {list(a.shape)} and w {list(w.shape)}: the summed axes differ")
    _vector(a_scale, "a_scale", (rows,), torch.float32, device)
    if out is None:
        out_dtype = out_dtype or torch.bfloat16
        if out_dtype not in TYPE_CODES:
            raise ValueError(f"out_dtype must be one of {FLOATS}")
        y, ldo = torch.empty_strided((rows, n), (n, 1), dtype=out_dtype, device=device), n
    else:
        y = _output(out, (rows, n), FLOATS, out_dtype, device,
                    (a, w, a_scale, w_scale) if ends is None else (a, w, a_scale, w_scale, ends))
        ldo = _ldo(y)
    ldw = _row_stride(ldw, n, k, 1)
    _launch(device, "b2m_int8_mm", a.data_ptr(), a_scale.data_ptr(), rows, _row_stride(lda, rows, k, 1), w.data_ptr(),
            w_scale.data_ptr(), experts, n, k, ldw, w_stride if experts > 1 else n * ldw,
            None if ends is None else ends.data_ptr(), y.data_ptr(), ldo, TYPE_CODES[y.dtype], out is None,
            None if status is None else _status_word(status, device))
    return y


def int8_mm(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
            out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
            status: torch.Tensor | None = None) -> torch.Tensor:
    """8-bit integer product with scales for each token and channel: ``y = (a @ w.T) * a_scale[:, None] * w_scale``.

    a int8 [M, K], w int8 [N, K] (``quant_int8`` of the activations and of the weights), a_scale fp32 [M], w_scale
    fp32 [N] -> [M, N] in bf16 (default), fp16 or fp32.  The integer sums are exact (K <= 131071); rows of a and w
    are a multiple of 16 bytes apart and 16-byte aligned.  ``status`` (``new_status``) records a wait that ran out of
    its limit and left the output unfinished.  Not differentiable: scales that require gradients are refused."""
    _cuda(a, "a")
    ldw, _ = _operand(w, "w", 2, torch.int8, a.device)
    n, k = w.shape
    _vector(w_scale, "w_scale", (n,), torch.float32, a.device)
    return _int8(a, a_scale, w, w_scale, 1, n, k, 0, ldw, None, out, out_dtype, status)


def int8_grouped_mm(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                    ends: torch.Tensor, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                    status: torch.Tensor | None = None) -> torch.Tensor:
    """``int8_mm`` over expert segments: a int8 [T, K], w int8 [E, N, K], a_scale fp32 [T], w_scale fp32 [E, N], ends
    int32 [E] -> [T, N]; ends, status and the rows behind ``ends[-1]`` as in ``grouped_mm``."""
    _cuda(a, "a")
    w_stride, ldw, _ = _operand(w, "w", 3, torch.int8, a.device)
    experts, n, k = w.shape
    _vector(ends, "ends", (experts,), torch.int32, a.device)
    _vector(w_scale, "w_scale", (experts, n), torch.float32, a.device)
    return _int8(a, a_scale, w, w_scale, experts, n, k, w_stride, ldw, ends, out, out_dtype, status)
