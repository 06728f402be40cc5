"""Python entry to the kernels over paged caches (eb_paged_append / eb_paged_attention).

Many sequences at once, each with a length of its own.  A packed batch: rows starts[b] to starts[b + 1] - 1 of the
activations are the new tokens of sequence b, lengths[b] counts its positions in the cache with them, and position p lies
in slot p mod page_size of page tables[b, p // page_size].  Pools are [pages, kv_heads, page_size, head_dim], in the
activations' type or torch.float8_e4m3fn with fp32 scales [pages, kv_heads] (value = code * scale).  starts, lengths and
tables are int32 on the device; a captured call may be replayed with other contents, within most_new new tokens per
sequence and most_length positions."""
import torch

from ._lib import lib, check, dtype_code, ptr, stream_ptr, require_cuda

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


def _one_device(what, *tensors):
    require_cuda(*tensors)
    here = torch.cuda.current_device()
    if any(t is not None and t.device.index != here for t in tensors):
        raise RuntimeError(f"{what}: all tensors must be on the current device (cuda:{here})")


def _rows(what, t, width, dtype):
    if t.dim() != 2 or t.stride(1) != 1 or t.shape[1] != width or t.dtype != dtype or (t.shape[0] > 1 and t.stride(0) < width):
        raise RuntimeError(f"{what}: rows of {width} contiguous columns of {dtype} required, not {tuple(t.shape)} of {t.dtype}")
    return t.stride(0) if t.shape[0] > 1 else width


def _cache(what, dtype, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale):
    """Checks pools and batch; returns (kv_heads, head_dim, arguments from `pages` on to `batch`)."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or not k_pages.is_contiguous() or not v_pages.is_contiguous():
        raise RuntimeError(f"{what}: pools are contiguous [pages, kv_heads, page_size, head_dim], alike for keys and values")
    pages, kv_heads, page_size, head_dim = k_pages.shape
    held = torch.float8_e4m3fn if k_scale is not None else dtype
    if k_pages.dtype != held or v_pages.dtype != held:
        raise RuntimeError(f"{what}: pools of {held} required" + ("" if k_scale is not None else " (8-bit pools go with scales)"))
    if (k_scale is None) != (v_scale is None) or any(s is not None and (s.dtype != torch.float32 or tuple(s.shape) != (pages, kv_heads) or not s.is_contiguous())
                                                     for s in (k_scale, v_scale)):
        raise RuntimeError(f"{what}: scales are contiguous fp32 [pages, kv_heads], for keys and for values")
    if any(t.dtype != torch.int32 for t in (tables, starts, lengths)) or tables.dim() != 2 or tables.stride(1) != 1 or lengths.shape != tables.shape[:1] or tuple(
            starts.shape) != (tables.shape[0] + 1,) or not starts.is_contiguous() or not lengths.is_contiguous():
        raise RuntimeError(f"{what}: int32 tables [batch, pages], starts [batch + 1] and lengths [batch] required")
    if tables.shape[0] == 0 or tables.shape[1] == 0 or (tables.shape[0] > 1 and tables.stride(0) < tables.shape[1]):
        raise RuntimeError(f"{what}: tables of one or more rows and columns required")
    return kv_heads, head_dim, (pages, page_size, ptr(tables), tables.stride(0) if tables.shape[0] > 1 else tables.shape[1], tables.shape[1], ptr(starts),
                                ptr(lengths), tables.shape[0])


def paged_append(q, k, v, k_pages, v_pages, tables, starts, lengths, most_new, freq=None, k_scale=None, v_scale=None, q_out=None):
    """New keys and values k, v [rows, kv_heads*head_dim] to their pages; freq (fp32: angle per position of each leading pair of
    neighbouring dimensions): queries q [rows, heads*head_dim] and keys are turned on the way.  q, k and v may be column
    ranges of one projection.  Returns the turned queries (in q_out, which may be q, or a new tensor; without freq: q itself
    unless q_out is given).  k_scale / v_scale belong to 8-bit pools and are updated: a page's scale grows to what its largest
    value needs, and the codes that it holds already are rounded to the new one."""
    _one_device("paged_append", q, k, v, k_pages, v_pages, tables, starts, lengths, freq, k_scale, v_scale, q_out)
    kv_heads, head_dim, where = _cache("paged_append", q.dtype, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale)
    rows = q.shape[0]
    if q.dim() != 2 or q.shape[1] % (kv_heads * head_dim) or k.shape[0] != rows or v.shape[0] != rows:
        raise RuntimeError("paged_append: one row of q, k and v per token, query heads in equal groups")
    ldq, ldk, ldv = (_rows("paged_append", t, w, q.dtype) for t, w in ((q, q.shape[1]), (k, kv_heads * head_dim), (v, kv_heads * head_dim)))
    if freq is not None and (freq.dtype != torch.float32 or freq.dim() != 1 or not freq.is_contiguous() or 2 * freq.numel() > head_dim):
        raise RuntimeError("paged_append: frequencies are fp32, one for each leading pair of a head")
    if freq is not None and q_out is None:
        q_out = torch.empty((rows, q.shape[1]), dtype=q.dtype, device=q.device)
    ldo = _rows("paged_append", q_out, q.shape[1], q.dtype) if q_out is not None else 0
    if q_out is not None and q_out.shape[0] != rows:
        raise RuntimeError("paged_append: one row of q_out per token")
    check(lib().eb_paged_append(ptr(q), ldq, ptr(k), ldk, ptr(v), ldv, ptr(q_out), ldo, rows, q.shape[1] // head_dim, kv_heads, head_dim, ptr(freq),
                                freq.numel() if freq is not None else 0, ptr(k_pages), ptr(v_pages), ptr(k_scale), ptr(v_scale), *where, int(most_new),
                                dtype_code(q.dtype), stream_ptr()), "paged_append")
    return q if q_out is None else q_out


def paged_attention(q, k_pages, v_pages, tables, starts, lengths, most_new, most_length=None, scale=None, window=0, k_scale=None, v_scale=None, out=None):
    """Causal attention of the new tokens q [rows, heads*head_dim] over their sequences' pages, which hold the new keys and values
    already: single tokens, a few per sequence, prompts and chunks of prompts, or all of them in one batch.  window > 0:
    the row at position p sees the positions above p - window only.  most_length: no sequence is longer (None: what the
    tables address).  Returns out [rows, heads*head_dim]; rows behind the last sequence are left as they are."""
    _one_device("paged_attention", q, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale, out)
    kv_heads, head_dim, where = _cache("paged_attention", q.dtype, k_pages, v_pages, tables, starts, lengths, k_scale, v_scale)
    if q.dim() != 2 or q.shape[1] % (kv_heads * head_dim):
        raise RuntimeError("paged_attention: q is [rows, heads*head_dim], query heads in equal groups")
    rows, heads, batch = q.shape[0], q.shape[1] // head_dim, tables.shape[0]
    ldq = _rows("paged_attention", q, q.shape[1], q.dtype)
    if out is None:
        out = torch.empty((rows, q.shape[1]), dtype=q.dtype, device=q.device)
    ldo = _rows("paged_attention", out, q.shape[1], q.dtype)
    if out.shape[0] != rows:
        raise RuntimeError("paged_attention: one row of out per row of q")
    reach = tables.shape[1] * k_pages.shape[2]
    most_length = reach if most_length is None else min(int(most_length), reach)
    most_new, window = min(int(most_new), rows), 0 if int(window) >= reach else int(window)
    nbytes = lib().eb_paged_attention_scratch_bytes(batch, heads, kv_heads, head_dim, most_new, most_length, window)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None       # (of this call: captured calls share none)
    check(lib().eb_paged_attention(ptr(q), ldq, ptr(out), ldo, rows, heads, kv_heads, head_dim, ptr(k_pages), ptr(v_pages), ptr(k_scale), ptr(v_scale), *where,
                                   most_new, most_length, window, float(head_dim ** -0.5 if scale is None else scale), dtype_code(q.dtype),
                                   ptr(scratch), nbytes, stream_ptr()), "paged_attention", launches=2 if nbytes else 1)
    return out
