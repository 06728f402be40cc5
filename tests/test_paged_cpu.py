"""Paged caches: what is refused before anything runs."""
import ctypes

import pytest
import torch

from energonai_b200 import _lib
from energonai_b200.paged import page_pools, paged_append, paged_attention, paged_batch


def test_a_batch_is_checked_on_the_host():
    ok = dict(new=[1, 3], lengths=[17, 3], tables=[[0, 5], [2]], pages=6, page_size=16, device="cpu")
    tables, starts, lengths, most_new, most_length = paged_batch(**ok)
    assert tables.tolist() == [[0, 5], [2, -1]] and starts.tolist() == [0, 1, 4] and lengths.tolist() == [17, 3] and (most_new, most_length) == (3, 17)
    for change, words in ((dict(new=[1]), "one entry"), (dict(new=[18, 3]), "new tokens"), (dict(new=[-1, 3]), "new tokens"), (dict(lengths=[33, 3]), "positions and"),
                          (dict(tables=[[0, 6], [2]]), "outside"), (dict(tables=[[0, -1], [2]]), "outside"), (dict(tables=[[5, 5], [2]]), "twice"),
                          (dict(tables=[[0, 5], [5]]), "write to page 5"), (dict(tables=[[2, 5], [2]]), "another one writes")):
        with pytest.raises(RuntimeError, match=words):
            paged_batch(**{**ok, **change})
    # a prefix that both only read may be shared, pages behind the last position may be anything of the pool
    paged_batch([1, 1], [17, 18], [[0, 5], [0, 2, 5]], 6, 16, device="cpu")
    # nothing new: nothing is written
    paged_batch([0, 0], [17, 18], [[0, 5], [0, 5]], 6, 16, device="cpu")


def test_pools_have_sizes_that_the_kernels_take():
    k, v, ks, vs = page_pools(3, 16, 2, 64, torch.float8_e4m3fn, device="cpu")
    assert k.shape == (3, 2, 16, 64) and v.dtype == torch.float8_e4m3fn and ks.shape == (3, 2) and vs.dtype == torch.float32
    assert page_pools(3, 16, 2, 64, torch.float16, device="cpu")[2:] == (None, None)
    for page, dim in ((8, 64), (24, 64), (16, 80)):
        with pytest.raises(RuntimeError):
            page_pools(3, page, 2, dim, torch.float16, device="cpu")


def test_cpu_tensors_are_rejected():
    k, v, _, _ = page_pools(3, 16, 2, 64, torch.float16, device="cpu")
    tables, starts, lengths, most_new, _ = paged_batch([1], [1], [[0]], 3, 16, device="cpu")
    q = torch.zeros(1, 256, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_append(q, q[:, :128], q[:, :128], k, v, tables, starts, lengths, most_new)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(q, k, v, tables, starts, lengths, most_new)


FAKE = 1 << 20                 # an aligned address that nothing is read from: every call below is refused before a launch


class Paged(ctypes.Structure):
    """struct eb_paged of the header."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k_pages", "v_pages", "k_scale", "v_scale", "tables", "starts", "lengths")] + [("table_ld", ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ("pages", "page_size", "kv_heads", "head_dim", "table_cols", "batch", "most_new", "most_length", "dtype", "reserved")]


def cache_of(a):
    names = [n for n, _ in Paged._fields_]
    return Paged(**{n: a.pop(n) for n in names if n in a}), a


def append_call(**change):
    a = dict(q=FAKE, ldq=512, k=FAKE, ldk=256, v=FAKE, ldv=256, q_out=FAKE, ldo=512, rows=4, heads=8, kv_heads=4, head_dim=64, freq=FAKE, pairs=32, k_pages=FAKE,
             v_pages=FAKE, k_scale=FAKE, v_scale=FAKE, pages=9, page_size=16, tables=FAKE, table_ld=3, table_cols=3, starts=FAKE, lengths=FAKE, batch=2, most_new=4,
             most_length=48, dtype=_lib.F16, stream=None)
    a.update(change)
    cache, a = cache_of(a)
    return _lib.lib().eb_paged_append(ctypes.addressof(cache), *a.values())


@pytest.mark.parametrize("change,words", [(dict(k=None), "null"), (dict(tables=None), "null"), (dict(dtype=_lib.F32), "fp16 or bf16"), (dict(head_dim=80), "head_dim 80"),
                                          (dict(page_size=24), "pages of 24"), (dict(kv_heads=3), "do not share"), (dict(v_scale=None), "scales"), (dict(pairs=33), "33 pairs"),
                                          (dict(freq=None), "pairs"), (dict(ldk=252), "strides"), (dict(ldk=260), "multiples of 8"), (dict(k=FAKE + 8), "16-byte"),
                                          (dict(table_ld=2), "bad sizes"), (dict(batch=65536), "bad sizes"), (dict(pages=0), "bad sizes"), (dict(most_new=-1), "at most -1"),
                                          (dict(table_cols=1 << 27, table_ld=1 << 27), "2^30")])
def test_append_refuses(change, words):
    assert append_call(**change) == -1 and words in _lib.last_error()


def attention_call(**change):
    a = dict(q=FAKE, ldq=512, out=FAKE, ldo=512, rows=4, heads=8, window=0, scale=0.125, kv_heads=4, head_dim=64, k_pages=FAKE, v_pages=FAKE, k_scale=None, v_scale=None, pages=9, page_size=16,
             tables=FAKE, table_ld=300, table_cols=300, starts=FAKE, lengths=FAKE, batch=2, most_new=4, most_length=4800, dtype=_lib.F16,
             scratch=FAKE, scratch_bytes=1 << 30, stream=None)
    a.update(change)
    cache, a = cache_of(a)
    return _lib.lib().eb_paged_attention(ctypes.addressof(cache), *a.values())


@pytest.mark.parametrize("change,words", [(dict(q=None), "null"), (dict(out=None), "null"), (dict(dtype=_lib.F32), "fp16 or bf16"), (dict(head_dim=96), "head_dim 96"),
                                          (dict(page_size=256), "pages of 256"), (dict(kv_heads=3), "do not share"), (dict(k_scale=FAKE), "scales"), (dict(scale=0.0), "positive"),
                                          (dict(scale=float("nan")), "positive"), (dict(window=-1), "window -1"), (dict(most_length=0), "most_length 0"), (dict(ldq=504), "strides"),
                                          (dict(ldo=516), "strides"), (dict(q=FAKE + 2), "16-byte"), (dict(scratch=None), "scratch"), (dict(scratch_bytes=64), "scratch")])
def test_attention_refuses(change, words):
    assert attention_call(**change) == -1 and words in _lib.last_error()


def test_empty_batches_are_accepted():
    assert append_call(rows=0) == 0 and append_call(batch=0) == 0 and append_call(most_new=0) == 0
    assert attention_call(rows=0) == 0 and attention_call(batch=0) == 0
    assert _lib.lib().eb_paged_attention_scratch_bytes(0, 8, 4, 64, 0, 1, 100, 0) == 0


def test_scratch_grows_with_the_splits():
    need = _lib.lib().eb_paged_attention_scratch_bytes
    assert need(1, 8, 8, 128, 0, 1, 64, 0) == 0                              # one CTA per head sees all keys
    assert need(1, 8, 8, 128, 0, 1, 100000, 0) > 0
    assert need(1, 8, 8, 128, 0, 1, 100000, 128) == 0                        # a window is short
    assert ctypes.sizeof(ctypes.c_size_t) == 8


def test_the_cache_struct_matches_the_header(tmp_path):
    """The bytes that the Python entry packs, and the structure above, have the size and field offsets that a C compiler gives the declaration."""
    import shutil
    import subprocess
    from energonai_b200 import paged
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    names = [n for n, _ in Paged._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(['#include <stdio.h>', '#include <stddef.h>', f'#include "{_lib.HEADER}"', 'int main(void) {', '  printf("%zu\\n", sizeof(eb_paged));']
                             + [f'  printf("%zu\\n", offsetof(eb_paged, {n}));' for n in names] + ['  return 0;', '}']))
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
    size, *offsets = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert ctypes.sizeof(Paged) == size == paged._paged.size
    assert [getattr(Paged, n).offset for n in names] == offsets
    packed = Paged.from_buffer_copy(paged._paged.pack(*range(1, len(names) + 1)))
    assert [getattr(packed, n) for n in names] == list(range(1, len(names) + 1))


def test_unknown_flags_are_refused():
    for call in (append_call, attention_call):
        assert call(reserved=2) == -1 and "flag bits" in _lib.last_error()


def test_scratch_is_bounded():
    """However many sequences a call brings and whatever the tables address: prompts beside many sequences, and steps of very long tables."""
    need = _lib.lib().eb_paged_attention_scratch_bytes
    for batch, heads, kv_heads, most_new, reach in ((64, 32, 8, 1024, 131072), (128, 40, 40, 1024, 131072), (128, 40, 40, 1, 131072), (64, 40, 40, 1, 1 << 20), (1024, 8, 8, 3, 131072),
                                                    (60000, 64, 8, 100, 1 << 24), (1, 128, 1, 1, (1 << 30) - 128)):
        for dim in (64, 128):
            # (the prompt form splits only what does not fill one wave)
            assert need(batch, heads, kv_heads, dim, 1, most_new, reach, 0) <= (256 + 20) << 20, (batch, heads, kv_heads, most_new, reach)
    assert need(1, 32, 8, 128, 1, 1, 131072, 0) > 0 and need(16, 32, 8, 128, 1, 100, 131072, 0) > 0


def test_sizes_that_no_call_takes_are_refused_by_name():
    """... and not by whatever they break on the way to the kernels."""
    from energonai_b200.paged import _cache
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    pools = lambda *shape: [torch.zeros(shape, dtype=torch.float16) for _ in range(2)]

    def call(pool=(3, 2, 16, 64), cols=2, batch=1, most_new=1, most_length=None):
        k, v = pools(*pool)
        return _cache("it", torch.float16, k, v, torch.empty((batch, cols), dtype=torch.int32), i32(batch + 1), i32(batch), None, None, most_new, most_length, False)

    assert call()[:3] == (2, 64, 32)
    for bad, words in ((dict(pool=(3, 0, 16, 64)), "pools of pages"), (dict(pool=(0, 2, 16, 64)), "pools of pages"), (dict(pool=(3, 2, 24, 64)), "pools of pages"),
                       (dict(pool=(3, 2, 16, 80)), "pools of pages"), (dict(cols=1 << 26), "2\\^30"), (dict(batch=1 << 16), "65535"), (dict(most_new=-1), "negative"),
                       (dict(most_length=-5), "negative"), (dict(cols=0), "one or more rows")):
        with pytest.raises(RuntimeError, match=words):
            call(**bad)
