"""Python entry to the kernels over paged caches (eb_paged_append / eb_paged_attention).

Many sequences at once, each with a length of its own.  A packed batch: rows starts[b] to starts[b + 1] - 1 of the
activations are the new tokens of sequence b, lengths[b] counts its positions in the cache with them, and position p lies
in slot p mod page_size of page tables[b, p // page_size].  Pools are [pages, kv_heads, page_size, head_dim], in the
activations' type or torch.float8_e4m3fn with fp32 scales [pages, kv_heads] (value = code * scale, scales not negative).  starts, lengths and
tables are int32 on the device; a captured call may be replayed with other contents, within most_new new tokens per
sequence and most_length positions."""
import functools
import struct

import torch

from ._lib import lib, check, dtype_code, require_cuda

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


def page_pools(pages, page_size, kv_heads, head_dim, dtype, device="cuda"):
    """New pools of a layer: (k_pages, v_pages, k_scale, v_scale); dtype torch.float8_e4m3fn: 8 bits with scales (else None)."""
    if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
        raise RuntimeError(f"page_pools: pages of {PAGE_SIZES} positions and heads of {HEAD_DIMS}")
    pools = [torch.zeros((pages, kv_heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(2)]
    scales = [torch.ones((pages, kv_heads), dtype=torch.float32, device=device) if dtype == torch.float8_e4m3fn else None for _ in range(2)]
    return (*pools, *scales)


def paged_batch(new, lengths, tables, pages, page_size, device="cuda"):
    """Checks a batch given as lists (new tokens, positions with them, pages of each sequence) and returns (tables, starts,
    lengths, most_new, most_length) for the functions below."""
    if not len(new) == len(lengths) == len(tables) or not new:
        raise RuntimeError("paged_batch: one entry per sequence")
    written = {}
    for b, (n, length, table) in enumerate(zip(new, lengths, tables)):
        if not 0 <= n <= length:
            raise RuntimeError(f"paged_batch: sequence {b} has {n} new tokens among {length} positions")
        if len(table) * page_size < length:
            raise RuntimeError(f"paged_batch: sequence {b} has {length} positions and {len(table)} pages of {page_size}")
        if any(not 0 <= p < pages for p in table):
            raise RuntimeError(f"paged_batch: sequence {b} names a page outside of the pool of {pages}")
        last = -(-length // page_size)
        if len(set(table[:last])) < last:
            raise RuntimeError(f"paged_batch: sequence {b} names a page twice")
        for p in table[(length - n) // page_size:last] if n else ():
            if written.setdefault(p, b) != b:
                raise RuntimeError(f"paged_batch: sequences {written[p]} and {b} write to page {p}")
    for b, (n, length, table) in enumerate(zip(new, lengths, tables)):
        if any(written.get(p, b) != b for p in table[:-(-length // page_size)]):
            raise RuntimeError(f"paged_batch: sequence {b} reads a page that another one writes")
    cols = max(1, max(len(t) for t in tables))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    return i32([list(t) + [-1] * (cols - len(t)) for t in tables]), i32(starts), i32(list(lengths)), max(new), max(1, max(lengths))


_device_here = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _one_device(what, *tensors):
    """All tensors (or None) are on the current device; returns its number."""
    here = None
    for t in tensors:
        if t is not None:
            on = t.get_device()
            if on != here:
                if here is not None or on < 0 or on != _device_here():
                    require_cuda(*tensors)
                    raise RuntimeError(f"{what}: all tensors must be on the current device (cuda:{_device_here()})")
                here = on
    return here


def _rows(what, t, width, dtype):
    """Row stride of [rows, width]."""
    shape = t.shape
    if len(shape) == 2 and shape[1] == width and t.dtype is dtype:
        ld, one = t.stride()
        if one == 1 or width == 1:
            if shape[0] <= 1:
                return width
            if ld >= width:
                return ld
    raise RuntimeError(f"{what}: rows of {width} contiguous columns of {dtype} required, not {tuple(shape)} of {t.dtype}")


def _new_like(q, most_new):
    """Rows for the results of q, contiguous as rows of q are; the kernel clears those of no sequence, unless nothing is announced."""
    return torch.empty_like(q) if most_new else torch.zeros_like(q)


# struct eb_paged of the header
_paged = struct.Struct("@7Pq10i")


def _cache(what, dtype, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale, most_new, most_length, clear):
    """Checks pools and batch; returns (kv_heads, head_dim, positions that the tables address, struct eb_paged)."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or not k_pages.is_contiguous() or not v_pages.is_contiguous():
        raise RuntimeError(f"{what}: pools are contiguous [pages, kv_heads, page_size, head_dim], alike for keys and values")
    pages, kv_heads, page_size, head_dim = shape
    if not 0 < pages < 1 << 31 or not 0 < kv_heads < 1 << 31 or page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
        raise RuntimeError(f"{what}: pools of pages of {PAGE_SIZES} positions and heads of {HEAD_DIMS} required, not {tuple(shape)}")
    if k_scale is None and v_scale is None:
        held, ks, vs = dtype, 0, 0
    else:
        held = torch.float8_e4m3fn
        per_block = shape[:2]
        if k_scale is None or v_scale is None or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32 or k_scale.shape != per_block or (
                v_scale.shape != per_block) or not k_scale.is_contiguous() or not v_scale.is_contiguous():
            raise RuntimeError(f"{what}: scales are contiguous fp32 [pages, kv_heads], for keys and for values")
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    if k_pages.dtype is not held or v_pages.dtype is not held:
        raise RuntimeError(f"{what}: pools of {held} required" + ("" if ks else " (8-bit pools go with scales)"))
    i32, of = torch.int32, tables.shape
    if tables.dtype is not i32 or starts.dtype is not i32 or lengths.dtype is not i32 or len(of) != 2 or lengths.shape != of[:1] or starts.shape != (
            of[0] + 1,) or not starts.is_contiguous() or not lengths.is_contiguous():
        raise RuntimeError(f"{what}: int32 tables [batch, pages], starts [batch + 1] and lengths [batch] required")
    batch, cols = of
    ld, one = tables.stride()
    if batch == 1:
        ld = cols
    if batch == 0 or cols == 0 or (one != 1 and cols > 1) or ld < cols:
        raise RuntimeError(f"{what}: int32 tables of one or more rows of contiguous columns required")
    reach = cols * page_size
    if reach >= 1 << 30 or batch >= 1 << 16:
        raise RuntimeError(f"{what}: a batch of {batch} sequences whose tables address {reach} positions exceeds 65535, or 2^30")
    if not 0 <= int(most_new) or (most_length is not None and not 0 <= int(most_length)):
        raise RuntimeError(f"{what}: negative limits (most_new {most_new}, most_length {most_length})")
    most_length = reach if most_length is None else min(int(most_length), reach)
    return kv_heads, head_dim, most_length, _paged.pack(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, tables.data_ptr(), starts.data_ptr(), lengths.data_ptr(), ld, pages,
                                                        page_size, kv_heads, head_dim, cols, batch, min(int(most_new), (1 << 31) - 1), most_length, dtype_code(dtype), 1 if clear else 0)


def paged_append(q, k, v, k_pages, v_pages, tables, starts, lengths, most_new, freq=None, k_scale=None, v_scale=None, q_out=None):
    """New keys and values k, v [rows, kv_heads*head_dim] to their pages; freq (fp32: angle per position of each leading pair of
    neighbouring dimensions): queries q [rows, heads*head_dim] and keys are turned on the way.  q, k and v may be column
    ranges of one projection.  Returns the turned queries (in q_out, which may be q, or a new tensor; without freq: q itself
    unless q_out is given).  Rows of no sequence, and those behind a sequence's first most_new, are zeros in a new tensor and left as they are in
    q_out.  k_scale / v_scale belong to 8-bit pools and are updated: a page's scale grows to what its largest
    value needs, and the codes that it holds already are rounded to the new one."""
    device = _one_device("paged_append", q, k, v, k_pages, v_pages, tables, starts, lengths, freq, k_scale, v_scale, q_out)
    dtype = q.dtype
    kv_heads, head_dim, _, cache = _cache("paged_append", dtype, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale, most_new, None, q_out is None)
    shape, width = q.shape, kv_heads * head_dim
    if len(shape) != 2 or shape[1] % width or k.shape[0] != shape[0] or v.shape[0] != shape[0]:
        raise RuntimeError("paged_append: one row of q, k and v per token, query heads in equal groups")
    rows, columns = shape
    ldq, ldk, ldv = _rows("paged_append", q, columns, dtype), _rows("paged_append", k, width, dtype), _rows("paged_append", v, width, dtype)
    pairs = 0
    if freq is not None:
        pairs = freq.numel()
        if freq.dtype is not torch.float32 or freq.dim() != 1 or not freq.is_contiguous() or 2 * pairs > head_dim:
            raise RuntimeError("paged_append: frequencies are fp32, one for each leading pair of a head")
        if q_out is None:
            q_out = _new_like(q, most_new)
    ldo = 0
    if q_out is not None:
        ldo = _rows("paged_append", q_out, columns, dtype)
        if q_out.shape[0] != rows:
            raise RuntimeError("paged_append: one row of q_out per token")
    check(lib().eb_paged_append(cache, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, None if q_out is None else q_out.data_ptr(), ldo, rows,
                                columns // head_dim, None if freq is None else freq.data_ptr(), pairs, _stream_of(device)), "paged_append")
    return q if q_out is None else q_out


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(*sizes):
    return lib().eb_paged_attention_scratch_bytes(*sizes)


def paged_attention(q, k_pages, v_pages, tables, starts, lengths, most_new, most_length=None, scale=None, window=0, k_scale=None, v_scale=None, out=None):
    """Causal attention of the new tokens q [rows, heads*head_dim] over their sequences' pages, which hold the new keys and values
    already: single tokens, a few per sequence, prompts and chunks of prompts, or all of them in one batch.  window > 0:
    the row at position p sees the positions above p - window only.  What a row does not see may hold anything, a value that is not finite makes
    what sees it infinite or NaN.  most_length: no sequence is longer (None: what the
    tables address).  Returns out [rows, heads*head_dim], which may be q.  Rows of no sequence, and those behind a sequence's first most_new,
    are left as they are in an out that is given, and zeros in a new tensor."""
    device = _one_device("paged_attention", q, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale, out)
    dtype, shape = q.dtype, q.shape
    kv_heads, head_dim, most_length, cache = _cache("paged_attention", dtype, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale, most_new, most_length, out is None)
    if len(shape) != 2 or shape[1] % (kv_heads * head_dim):
        raise RuntimeError("paged_attention: q is [rows, heads*head_dim], query heads in equal groups")
    rows, columns = shape
    heads = columns // head_dim
    ldq = _rows("paged_attention", q, columns, dtype)
    if out is None:
        out = _new_like(q, most_new)
        ldo = columns
    else:
        ldo = _rows("paged_attention", out, columns, dtype)
        if out.shape[0] != rows:
            raise RuntimeError("paged_attention: one row of out per row of q")
    window = int(window)
    if window < 0:
        raise RuntimeError(f"paged_attention: a window of {window} positions")
    if window >= most_length:
        window = 0                                          # (every key is inside)
    nbytes = _scratch_bytes(tables.shape[0], heads, kv_heads, head_dim, k_scale is not None, min(int(most_new), rows), most_length, window)
    scratch = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None       # (of this call: captured calls share none)
    check(lib().eb_paged_attention(cache, q.data_ptr(), ldq, out.data_ptr(), ldo, rows, heads, window, float(head_dim ** -0.5 if scale is None else scale),
                                   None if scratch is None else scratch.data_ptr(), nbytes, _stream_of(device)), "paged_attention", launches=2 if nbytes else 1)
    return out
