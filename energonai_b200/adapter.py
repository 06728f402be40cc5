"""Python entry to the low-rank adapters of many requests (eb_adapter_delta) beside a shared projection."""
import functools

import torch

from ._lib import lib, check, dtype_code
from .gemm import gemm
from .paged import _one_device, _rows, _stream_of

MAX_RANK = 128


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(*sizes):
    return lib().eb_adapter_scratch_bytes(*sizes)


def adapter_delta(x, a, b, scales, index, starts, most_new):
    """What each row's adapter adds to a projection of x [rows, width]: scales[i] (x a[i].T) b[i].T, [rows, columns], with
    i = index[s] for the rows starts[s] to starts[s + 1] - 1 of sequence s (at most most_new).  a [adapters, rank, width], b
    [adapters, columns, rank], scales fp32 [adapters]; index int32 [batch], negative for none; starts int32 [batch + 1].  rank is
    a multiple of 8 up to MAX_RANK (smaller adapters are filled up with zeros).  Rows of no sequence, and
    those behind a sequence's first most_new, get zeros."""
    return _adapters("adapter_delta", x, a, b, scales, index, starts, most_new)


def _adapters(what, x, a, b, scales, index, starts, most_new, base=None, out=None):
    """adapter_delta, or what base() returns (fp32) and adapter_delta, added up and rounded once (to out, of the type of x)."""
    device = _one_device(what, x, a, b, scales, index, starts)
    dtype, shape, of, to = x.dtype, x.shape, a.shape, b.shape
    if len(of) != 3 or len(to) != 3 or len(shape) != 2 or of[0] != to[0] or of[1] != to[2] or of[2] != shape[1]:
        raise RuntimeError(f"{what}: x [rows, width], a [adapters, rank, width] and b [adapters, columns, rank] required")
    if a.dtype is not dtype or b.dtype is not dtype or not a.is_contiguous() or not b.is_contiguous():
        raise RuntimeError(f"{what}: adapters are contiguous and of the type of x")
    adapters, rank, width = of
    if scales.dtype is not torch.float32 or scales.shape != (adapters,) or not scales.is_contiguous():
        raise RuntimeError(f"{what}: one fp32 scale per adapter")
    batch = index.numel()
    if index.dtype is not torch.int32 or starts.dtype is not torch.int32 or index.dim() != 1 or starts.shape != (batch + 1,) or batch == 0 or not (
            index.is_contiguous() and starts.is_contiguous()):
        raise RuntimeError(f"{what}: int32 index [batch] and starts [batch + 1] required")
    rows, columns, most_new = shape[0], to[1], int(most_new)
    ldx = _rows(what, x, width, dtype)
    given, out = out, out if out is not None and out.stride(0) % 8 == 0 else x.new_empty((rows, columns))
    if most_new == 0:                                                    # (no row has an adapter)
        nothing = x.new_zeros((rows, columns)) if base is None else base().to(dtype)
        return nothing if given is None else given.copy_(nothing)
    nbytes = _scratch_bytes(rows, width, rank, batch, most_new)
    scratch = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None       # (of this call: captured calls share none)
    of, sequences = (x.data_ptr(), ldx, a.data_ptr()), (index.data_ptr(), starts.data_ptr())
    sizes = (rank, adapters, batch, most_new, dtype_code(dtype), None if scratch is None else scratch.data_ptr(), nbytes, _stream_of(device))
    to = (out.data_ptr(), _rows(what, out, columns, dtype), rows, width, columns)
    if base is None:
        check(lib().eb_adapter_delta(*of, b.data_ptr(), scales.data_ptr(), *sequences, *to, *sizes), what, launches=2)
        return out
    check(lib().eb_adapter_low(*of, *sequences, rows, width, *sizes), what)
    sums = base()
    check(lib().eb_adapter_add(b.data_ptr(), scales.data_ptr(), *sequences, sums.data_ptr(), columns, *to, *sizes), what)
    return out if given is None or given is out else given.copy_(out)      # (rows that do not begin on 16 bytes)


def adapter_product(x, w, a, b, scales, index, starts, most_new, bias=None, out=None, static_weight=False):
    """x @ w.T + bias for all rows, and beside it each sequence's adapter (adapter_delta), added to the fp32 sums: [rows, columns].
    Rows of no sequence, and those behind a sequence's first most_new, get the shared projection alone.  Calls on several streams and replayed graphs may overlap."""
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
    if x.dtype is torch.float16:                            # (the adapter's part alone may be beyond fp16)
        return _adapters("adapter_product", x, a, b, scales, index, starts, most_new,
                         lambda: gemm(x, w, bias=bias, out_dtype=torch.float32, static_weight=static_weight, overlap=True), out)
    return gemm(x, w, bias=bias, residual=adapter_delta(x, a, b, scales, index, starts, most_new), out=out, static_weight=static_weight, overlap=True)
