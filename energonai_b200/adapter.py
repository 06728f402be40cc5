"""Python entry to the low-rank adapters of many requests (eb_adapter_delta) beside a shared projection."""
import torch

from ._lib import lib, check, dtype_code, ptr, stream_ptr
from .gemm import gemm
from .paged import _one_device, _rows

MAX_RANK = 128


def adapter_delta(x, a, b, scales, index, starts, most_new):
    """What each row's adapter adds to a projection of x [rows, width]: scales[i] (x a[i].T) b[i].T, [rows, columns], with
    i = index[s] for the rows starts[s] to starts[s + 1] - 1 of sequence s (at most most_new).  a [adapters, rank, width], b
    [adapters, columns, rank], scales fp32 [adapters]; index int32 [batch], negative for none; starts int32 [batch + 1].  rank is
    a multiple of 8 up to MAX_RANK (smaller adapters are filled up with zeros).  Rows behind the last sequence get zeros."""
    _one_device("adapter_delta", x, a, b, scales, index, starts)
    if a.dim() != 3 or b.dim() != 3 or x.dim() != 2 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or a.shape[2] != x.shape[1]:
        raise RuntimeError("adapter_delta: x [rows, width], a [adapters, rank, width] and b [adapters, columns, rank] required")
    if a.dtype != x.dtype or b.dtype != x.dtype or not a.is_contiguous() or not b.is_contiguous():
        raise RuntimeError("adapter_delta: adapters are contiguous and of the type of x")
    adapters, rank, width = a.shape
    if scales.dtype != torch.float32 or tuple(scales.shape) != (adapters,) or not scales.is_contiguous():
        raise RuntimeError("adapter_delta: one fp32 scale per adapter")
    if any(t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() for t in (index, starts)) or starts.numel() != index.numel() + 1 or index.numel() == 0:
        raise RuntimeError("adapter_delta: int32 index [batch] and starts [batch + 1] required")
    rows, columns, batch = x.shape[0], b.shape[1], index.numel()
    ldx = _rows("adapter_delta", x, width, x.dtype)
    delta = torch.empty((rows, columns), dtype=x.dtype, device=x.device)
    nbytes = lib().eb_adapter_scratch_bytes(rows, width, rank, batch, int(most_new))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None       # (of this call: captured calls share none)
    check(lib().eb_adapter_delta(ptr(x), ldx, ptr(a), ptr(b), ptr(scales), ptr(index), ptr(starts), ptr(delta), columns, rows, width, columns, rank, adapters,
                                 batch, int(most_new), dtype_code(x.dtype), ptr(scratch), nbytes, stream_ptr()), "adapter_delta", launches=2)
    return delta


def adapter_product(x, w, a, b, scales, index, starts, most_new, bias=None, out=None, static_weight=False):
    """x @ w.T + bias for all rows, and beside it each sequence's adapter (adapter_delta), added to the fp32 sums: [rows, columns].
    Rows behind the last sequence get the shared projection alone."""
    _one_device("adapter_product", w, bias, out)
    if w.dim() != 2 or w.shape != (b.shape[1], x.shape[1]) or w.dtype != x.dtype:
        raise RuntimeError("adapter_product: the shared weight is [columns, width] of the type of x")
    if bias is not None and (bias.dtype != x.dtype or bias.shape != w.shape[:1] or not bias.is_contiguous()):
        raise RuntimeError("adapter_product: the bias has the type of x and one entry per column")
    if out is not None:
        _rows("adapter_product", out, w.shape[0], x.dtype)
        if out.shape[0] != x.shape[0]:
            raise RuntimeError("adapter_product: one row of out per row of x")
    if x.shape[0] == 0:
        return torch.empty((0, w.shape[0]), dtype=x.dtype, device=x.device) if out is None else out
    return gemm(x, w, bias=bias, residual=adapter_delta(x, a, b, scales, index, starts, most_new), out=out, static_weight=static_weight)
