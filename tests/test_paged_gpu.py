"""Kernels over paged caches against the restatement in 64 bits."""
import math

import pytest
import torch

from paged_plain import E4M3, Case

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def close(got, want, tol, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    over = (got - want).abs() - tol
    assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} above the tolerance, at {int(over.flatten().argmax())}"


def frequencies(pairs):
    return 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))


def check_append(c, pairs, got, pools, scales):
    freq = frequencies(pairs).float() if pairs else None
    want = c.append(freq)
    n = c.starts[-1]
    close(got[:n], want[0][0][:n], want[0][1][:n], "queries")
    for i, name in ((0, "keys"), (1, "values")):
        value, tol, scale = want[1 + i]
        have = pools[i].double().cpu()
        if c.bits == 8:
            assert torch.equal(scales[i].cpu(), scale), name
            have = have * scale.double()[..., None, None]
        assert torch.equal(torch.isnan(have), torch.isnan(value)), name
        there = ~torch.isnan(value)
        assert bool(((have - value).abs()[there] <= tol[there]).all()), (name, float(((have - value).abs() - tol)[there].max()))


BATCHES = [([1], [0]), ([1, 1, 1, 1, 1], [0, 15, 16, 31, 300]), ([5, 0, 1, 37], [7, 9, 64, 0]), ([150, 3], [0, 130]), ([16], [16])]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("new,past", BATCHES)
@pytest.mark.parametrize("heads,kv_heads,dim,page,pairs", [(4, 4, 64, 16, 32), (6, 2, 128, 32, 64), (5, 1, 64, 128, 0), (3, 3, 128, 64, 11)])
def test_append(new, past, heads, kv_heads, dim, page, pairs, bits, dtype):
    from energonai_b200.paged import paged_append
    c = Case(new, past, heads, kv_heads, dim, page, dtype, bits, seed=sum(new) + dim)
    (q, k, v), pools, scales, (tables, starts, lengths, most_new) = c.device()
    freq = frequencies(pairs).float().cuda() if pairs else None
    got = paged_append(q, k, v, *pools, tables, starts, lengths, most_new, freq=freq, k_scale=scales[0], v_scale=scales[1])
    assert (got is q) == (pairs == 0)
    check_append(c, pairs, got, pools, scales)


def test_append_takes_columns_of_a_projection_and_leaves_other_rows():
    from energonai_b200.paged import paged_append
    c = Case([4, 1], [3, 40], 4, 2, 64, 16, BF16, 8, seed=5, pad_rows=3)
    (q, k, v), pools, scales, (tables, starts, lengths, most_new) = c.device(bad=1 << 30)
    proj = torch.cat([q, k, v, torch.zeros_like(q)], 1)
    q, k, v = proj[:, :256], proj[:, 256:384], proj[:, 384:512]
    before = proj.clone()
    got = paged_append(q, k, v, *pools, tables, starts, lengths, most_new, freq=frequencies(32).float().cuda(), k_scale=scales[0], v_scale=scales[1], q_out=q)
    assert got.data_ptr() == proj.data_ptr()
    check_append(c, 32, got, pools, scales)
    assert torch.equal(proj[:, 256:], before[:, 256:]) and torch.equal(proj[5:], before[5:])


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("most_new", [1, 3, 16, 17])
def test_append_leaves_out_rows_behind_the_announced_ones(most_new, bits):
    """A sequence that brings more rows than announced loses the others, and no memory is touched for them."""
    from energonai_b200.paged import paged_append
    c = Case([40, 2], [0, 5], 4, 2, 128, 16, F16, bits, seed=4)
    (q, k, v), pools, scales, (tables, starts, lengths, _) = c.device()
    before = [p.clone() for p in pools]
    freq = frequencies(64).float().cuda()
    got = paged_append(q, k, v, *pools, tables, starts, lengths, most_new, freq=freq, k_scale=scales[0], v_scale=scales[1], q_out=torch.full_like(q, 7.0))
    whole, fresh = before, [None if x is None else x.clone() for x in c.device()[2]]
    want = paged_append(q, k, v, *whole, tables, starts, lengths, 40, freq=freq, k_scale=fresh[0], v_scale=fresh[1])
    n = min(most_new, 40)
    assert torch.equal(got[:n], want[:n]) and bool((got[n:40] == 7.0).all()) and torch.equal(got[40:40 + min(n, 2)], want[40:40 + min(n, 2)])
    last = c.pool[0][c.tables[0][2]].view(torch.uint8 if bits == 8 else torch.int16)                  # (rows 32 .. 39: announced by none of these)
    have = pools[0][c.tables[0][2]].view(last.dtype).cpu()
    assert torch.equal(have, last)


def test_append_far_positions():
    """The angle is taken in 64 bits: at position 2 million a 32-bit one would be off by 0.1."""
    from energonai_b200.paged import paged_append
    c = Case([2], [0], 2, 2, 128, 128, F16, 16, seed=3)
    far = 2_000_000 // 128 * 128
    (q, k, v), pools, scales, (_, starts, _, most_new) = c.device()
    tables = torch.full((1, far // 128 + 1), -1, dtype=torch.int32, device="cuda")
    tables[0, -1] = c.tables[0][0]
    lengths = torch.tensor([far + 2], dtype=torch.int32, device="cuda")
    got = paged_append(q, k, v, *pools, tables, starts, lengths, most_new, freq=frequencies(64).float().cuda())
    c.past, c.length = [far], [far + 2]
    x, slack = c.turned(c.q, frequencies(64).float())
    close(got, x.flatten(1), (2.0 ** -11 * (x.abs() + slack) + slack).flatten(1))
    x, slack = c.turned(c.k, frequencies(64).float())
    have = pools[0][c.tables[0][0], :, :2].transpose(0, 1)
    close(have, x, 2.0 ** -11 * (x.abs() + slack) + slack)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_eight_bit_pages_token_by_token(dtype):
    """A page's scale grows with its largest value, earlier codes follow; zeros, the smallest and the largest numbers, infinities
    and NaN."""
    from energonai_b200.paged import paged_append
    c = Case([1], [0], 1, 1, 64, 16, dtype, 8, seed=9)
    (q, k, v), pools, scales, (tables, starts, _, _) = c.device()
    big = float(torch.finfo(dtype).max)
    rows = [torch.zeros(64), torch.full((64,), 1e-6), torch.linspace(-3, 3, 64), torch.linspace(-40, 40, 64), torch.full((64,), big), torch.linspace(-1, 1, 64)]
    rows[3][5], rows[3][6], rows[3][7] = float("inf"), float("-inf"), float("nan")
    held = torch.zeros(0, 64, dtype=torch.float64)
    scale = 0.0
    for n, row in enumerate(rows):
        x = row.to(dtype)[None].cuda()
        lengths = torch.tensor([n + 1], dtype=torch.int32, device="cuda")
        paged_append(x, x, x, *pools, tables, starts, lengths, 1, k_scale=scales[0], v_scale=scales[1])
        x = x.double().cpu()
        x[~torch.isfinite(x)] = float("nan")
        m = float(x.nan_to_num(0).abs().max())
        need = 2.0 ** max(-100, math.ceil(math.log2(m / 448))) if m else 2.0 ** -100
        scale = need if n == 0 else max(scale, need)
        held = torch.cat([(held / scale).float().to(E4M3).double() * scale, (x / scale).float().to(E4M3).double() * scale])
        for i in (0, 1):
            assert float(scales[i][c.tables[0][0], 0]) == scale, n
            have = pools[i][c.tables[0][0], 0, :n + 1].double().cpu() * scale
            assert torch.equal(have.nan_to_num(7.0), held.nan_to_num(7.0)) and torch.equal(have.isnan(), held.isnan()), n


STEPS = [([1], [0]), ([1], [16]), ([1, 1, 1], [3, 4000, 1023]), ([1] * 17, list(range(0, 34, 2))), ([1, 0, 1], [700, 5, 31])]
FEW = [([2, 5, 1], [0, 100, 513]), ([16], [1]), ([7, 3], [0, 2047]), ([33], [0])]
HEADS = [(4, 4, 64), (2, 2, 128), (8, 2, 128), (7, 1, 64), (12, 1, 128), (10, 2, 128), (16, 1, 64), (17, 1, 128)]


@pytest.mark.parametrize("dtype,bits", [(F16, 16), (BF16, 16), (F16, 8), (BF16, 8)])
@pytest.mark.parametrize("new,past", STEPS + FEW)
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_attention_of_few_tokens(new, past, heads, kv_heads, dim, bits, dtype):
    from energonai_b200.paged import paged_attention
    page = (16, 32, 64, 128)[(heads + len(new)) % 4]
    c = Case(new, past, heads, kv_heads, dim, page, dtype, bits, seed=heads + sum(past))
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    for window in (0, 20) if max(past) < 2000 else (0, 700):
        got = paged_attention(q, *pools, tables, starts, lengths, most_new, max(c.length), window=window, k_scale=scales[0], v_scale=scales[1])
        close(got, *c.attention(window=window, prompt=64 * kv_heads // heads), f"window {window}")


PROMPTS = [([65], [0]), ([300, 64], [0, 5]), ([257, 1, 0, 90], [200, 1000, 3, 16]), ([1, 700], [0, 1]), ([128, 256, 129], [128, 0, 1]), ([70], [5000])]


@pytest.mark.parametrize("dtype,bits", [(F16, 16), (BF16, 16), (F16, 8), (BF16, 8)])
@pytest.mark.parametrize("new,past", PROMPTS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (2, 2, 128), (8, 2, 128), (7, 1, 64), (6, 2, 128)])
def test_attention_of_prompts(new, past, heads, kv_heads, dim, bits, dtype):
    from energonai_b200.gemm import device_status
    from energonai_b200.paged import paged_attention
    page = (16, 32, 64, 128)[(heads + len(new) + max(new)) % 4]
    c = Case(new, past, heads, kv_heads, dim, page, dtype, bits, seed=heads + sum(past) + max(new))
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    for window in (0, 1, 50, 333):
        got = paged_attention(q, *pools, tables, starts, lengths, most_new, max(c.length), window=window, k_scale=scales[0], v_scale=scales[1])
        want, tol = c.attention(window=window, prompt=64 * kv_heads // heads)
        close(got, want, tol, f"window {window}")
    assert device_status()[0] == 0


@pytest.mark.parametrize("bits", [8, 16])
def test_prompt_pages_that_are_none(bits):
    """Keys of pages outside of the pool are not there for any row, in prompts too."""
    from energonai_b200.paged import paged_attention
    c = Case([200], [300], 2, 1, 128, 32, BF16, bits, seed=21)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device(bad=1 << 29)
    for at, bad in ((0, -1), (3, 1 << 30), (9, c.pages)):
        tables[0, at] = bad
    got = paged_attention(q, *pools, tables, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1])
    close(got, *c.attention(prompt=32, missing=(0, 3, 9)))


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (BF16, 8), (F16, 8)])
@pytest.mark.parametrize("magnitude", [1e-3, 30.0, 1e4])
def test_attention_magnitudes(magnitude, bits, dtype):
    """Scores from almost equal to one-sided, queries far above and below fp16's normal range in bf16."""
    from energonai_b200.paged import paged_attention
    c = Case([1, 3, 90], [100, 50, 40], 4, 2, 128, 16, dtype, bits, seed=4, magnitude=magnitude if dtype == BF16 or magnitude < 1e4 else 3e3)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    scale = 1 / magnitude if magnitude > 100 else 0.3
    got = paged_attention(q, *pools, tables, starts, lengths, most_new, scale=scale, k_scale=scales[0], v_scale=scales[1])
    close(got, *c.attention(scale=scale, prompt=32))


def test_pages_of_very_different_scales():
    """Values of one page are 2^30 times those of another: rows that look at the small page only keep their precision."""
    from energonai_b200.paged import paged_attention
    c = Case([1], [31], 1, 1, 64, 16, F16, 8, seed=8)
    c.scale[1][c.tables[0][0]] *= 2.0 ** 30
    c.scale[0][:] = 2.0 ** -6
    c.pool[0] = torch.zeros_like(c.pool[0], dtype=torch.float32).to(E4M3)
    first, second = c.tables[0]
    c.pool[0][first] = torch.full((1, 16, 64), -448.0).to(E4M3)              # far below the keys of the second page
    c.q = torch.full_like(c.q, 4.0)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    got = paged_attention(q, *pools, tables, starts, lengths, most_new, scale=1.0, k_scale=scales[0], v_scale=scales[1])
    close(got, *c.attention(scale=1.0))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("least", [2.0 ** -100, 2.0 ** -40, 0.0])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (2, 2, 128, 32), (24, 1, 128, 16)])
def test_pages_of_tiny_values_keep_their_share_of_the_weights(heads, kv_heads, dim, page, least, dtype):
    """Every fifth page has values far smaller than the others' (or none): its keys take their weights from the others all the same."""
    from energonai_b200.paged import paged_attention
    c = Case([1, 70, 5, 2], [31, 0, 200, 9], heads, kv_heads, dim, page, dtype, 8, seed=heads)
    for page in [p for t in c.tables for p in t[::5]]:
        c.scale[1][page] = least
        if least < 2.0 ** -40:
            codes = c.pool[1][page].view(torch.uint8)
            codes[codes != 0x7f] = 0
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    close(paged_attention(q, *pools, tables, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1]), *c.attention())


def test_rows_without_keys_and_rows_behind_the_last_sequence():
    from energonai_b200.paged import paged_attention
    c = Case([1, 2], [40, 5], 4, 4, 64, 16, F16, 16, seed=2, pad_rows=4)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device(bad=1 << 29)
    tables[0] = -1                                                           # the first sequence has no pages at all
    out = torch.full_like(q, 3.0)
    paged_attention(q, *pools, tables, starts, lengths, most_new, out=out)
    want, tol = c.attention()
    assert not out[0].any()
    close(out[1:3], want[1:3], tol[1:3])
    assert bool((out[3:] == 3.0).all())


def test_strided_queries_and_output():
    from energonai_b200.paged import paged_attention
    c = Case([1, 4], [70, 9], 4, 2, 128, 32, BF16, 16, seed=6)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    wide, out = torch.zeros(5, 1024 + 8, dtype=BF16, device="cuda"), torch.zeros(5, 2048, dtype=BF16, device="cuda")
    wide[:, 8:520] = q
    got = paged_attention(wide[:, 8:520], *pools, tables, starts, lengths, most_new, out=out[:, 512:1024])
    close(got, *c.attention())
    assert not out[:, :512].any() and not out[:, 1024:].any()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("new,past", [([3, 1, 40, 2], [0, 300, 30, 5]), ([200, 1, 150, 90], [10, 3, 900, 0])])
def test_a_part_of_a_batch(new, past, bits):
    """The later sequences alone, out of tensors that hold them all: the rows in front of theirs stay as they are."""
    from energonai_b200.paged import paged_append, paged_attention
    c = Case(new, past, 6, 2, 128, 32, BF16, bits, seed=9, pad_rows=2)
    (q, k, v), pools, scales, (tables, starts, lengths, most_new) = c.device()
    freq = frequencies(64).float()
    some = (tables[1:], starts[1:], lengths[1:])
    want = c.append(freq)
    turned = paged_append(q, k, v, *pools, *some, most_new, freq=freq.cuda(), k_scale=scales[0], v_scale=scales[1], q_out=torch.full_like(q, 2.0))
    n, end = c.starts[1], c.starts[-1]
    close(turned[n:end], want[0][0][n:end], want[0][1][n:end])
    assert bool((turned[:n] == 2.0).all()) and bool((turned[end:] == 2.0).all())
    for i in (0, 1):                                                         # (the first sequence's pages: as before)
        first = torch.tensor(c.tables[0], dtype=torch.long)
        assert torch.equal(pools[i].cpu()[first].view(torch.uint8), c.pool[i][first].view(torch.uint8))
    out = paged_attention(q, *pools, *some, most_new, k_scale=scales[0], v_scale=scales[1], out=torch.full_like(q, 3.0))
    c.pool, c.scale = [p.cpu() for p in pools], [None if s is None else s.cpu() for s in scales]
    value, tol = c.attention(prompt=64 // 3)
    close(out[n:end], value[n:end], tol[n:end])
    assert bool((out[:n] == 3.0).all()) and bool((out[end:] == 3.0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("new,past,heads,kv_heads", [([1, 5, 2], [700, 30, 9], 8, 2), ([300, 1, 129], [0, 900, 60], 6, 2), ([80], [20000], 8, 8), ([130, 70], [5, 0], 10, 2)])
def test_in_place_over_the_queries(new, past, heads, kv_heads, bits, dtype):
    from energonai_b200.paged import paged_attention
    c = Case(new, past, heads, kv_heads, 64, 64, dtype, bits, seed=11)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    want = paged_attention(q, *pools, tables, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(paged_attention(q, *pools, tables, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1], out=q), want)


@pytest.mark.parametrize("bits", [8, 16])
def test_sequences_that_share_their_first_pages(bits):
    from energonai_b200.paged import paged_attention
    c = Case([1, 70, 3], [100, 40, 60], 4, 2, 64, 16, F16, bits, seed=12)
    for t in c.tables[1:]:
        t[:2] = c.tables[0][:2]
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    close(paged_attention(q, *pools, tables, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1]), *c.attention())


def test_results_do_not_depend_on_the_other_sequences():
    """A sequence gets the same bits alone and in a batch that is cut alike, and the same bits every time."""
    from energonai_b200.paged import paged_attention
    c = Case([1] * 8, [900, 3, 77, 1500, 64, 640, 1, 2000], 8, 2, 128, 16, BF16, 8, seed=1)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    kw = dict(k_scale=scales[0], v_scale=scales[1])
    a = paged_attention(q, *pools, tables, starts, lengths, 1, **kw)
    for _ in range(3):
        assert torch.equal(a, paged_attention(q, *pools, tables, starts, lengths, 1, **kw))


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("new,watched", [([1, 2, 1, 3, 1], (0, 3)), ([90, 1, 200, 5, 1], (0, 1, 2, 3))])
def test_a_sequence_does_not_depend_on_the_others(new, watched, bits):
    """The same bits whatever the other sequences bring, hold and are long, in a batch that is cut alike."""
    from energonai_b200.paged import paged_attention
    past = [9000, 8300, 30, 700, 5]
    c = Case(new, past, 8, 2, 128, 16, BF16, bits, seed=1)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    kw = dict(k_scale=scales[0], v_scale=scales[1])
    want = paged_attention(q, *pools, tables, starts, lengths, most_new, **kw)
    close(want, *c.attention(prompt=16))
    for b in watched:
        rows, mine = slice(c.starts[b], c.starts[b + 1]), torch.zeros(c.pages, dtype=torch.bool, device="cuda")
        mine[torch.tensor(c.tables[b], device="cuda")] = True
        other = [p.clone() for p in pools]
        for p in other:
            p.view(torch.uint8)[~mine] = 0x35
        zs = [None if s is None else torch.where(mine[:, None], s, 2.0 * s) for s in scales]
        q2, lengths2, tables2 = -q, torch.clamp(lengths - 3, min=1), tables.flip(1).contiguous()
        q2[rows], lengths2[b], tables2[b] = q[rows], lengths[b], tables[b]
        lengths2 = torch.maximum(lengths2, starts[1:] - starts[:-1])
        assert torch.equal(paged_attention(q2, *other, tables2, starts, lengths2, most_new, k_scale=zs[0], v_scale=zs[1])[rows], want[rows]), b
        # the others bring nothing: its rows alone, in the same places
        starts3 = torch.tensor([c.starts[b] if i <= b else c.starts[b + 1] for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        assert torch.equal(paged_attention(q2, *other, tables2, starts3, lengths2, most_new, k_scale=zs[0], v_scale=zs[1])[rows], want[rows]), b


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("new,past", [([1, 1], [40, 9]), ([3, 1, 40, 2], [0, 300, 30, 5]), ([200, 1, 150, 90], [10, 3, 900, 0]), ([1, 0, 1], [20000, 5, 7])])
def test_rows_of_no_sequence_of_new_tensors_are_zeros(new, past, bits):
    """In front of the first sequence and behind the last one, behind the announced rows, and of a sequence that is none: zeros where the call makes the
    tensor, nothing where the caller gives it."""
    from energonai_b200.paged import paged_append, paged_attention
    c = Case(new, past, 6, 2, 128, 32, BF16, bits, seed=9, pad_rows=5)
    (q, k, v), pools, scales, (tables, starts, lengths, most_new) = c.device()
    freq = frequencies(64).float().cuda()
    kw = dict(k_scale=scales[0], v_scale=scales[1])
    dirty = lambda: torch.full_like(q, float("nan"))                         # (what an output that is not written would hold)

    def both(tables, starts, lengths, most_new):
        dirty()
        turned = paged_append(q, k, v, *[p.clone() for p in pools], tables, starts, lengths, most_new, freq=freq, k_scale=None if bits == 16 else scales[0].clone(),
                              v_scale=None if bits == 16 else scales[1].clone())
        dirty()
        out = paged_attention(q, *pools, tables, starts, lengths, most_new, **kw)
        given = paged_attention(q, *pools, tables, starts, lengths, most_new, out=torch.full_like(q, 3.0), **kw)
        turned_given = paged_append(q, k, v, *[p.clone() for p in pools], tables, starts, lengths, most_new, freq=freq, k_scale=None if bits == 16 else scales[0].clone(),
                                    v_scale=None if bits == 16 else scales[1].clone(), q_out=torch.full_like(q, 3.0))
        return (turned, turned_given), (out, given)

    def check(pairs, none):
        for made, given in pairs:
            assert not made[none].any() and bool((given[none] == 3.0).all())
            assert torch.equal(made[~none], given[~none]) and bool(made[~none].isfinite().all())

    none = torch.zeros(c.rows, dtype=torch.bool, device="cuda")
    none[c.starts[-1]:] = True
    check(both(tables, starts, lengths, most_new), none)
    # the later sequences alone
    none[:c.starts[1]] = True
    check(both(tables[1:], starts[1:], lengths[1:], most_new), none)
    # a sequence with fewer positions than new tokens is none
    none[:c.starts[1]] = True
    wrong = lengths.clone()
    wrong[0] = new[0] - 1
    check(both(tables, starts, wrong, most_new), none)
    # fewer rows are announced than come
    if most_new > 2:
        few = most_new // 3
        none = torch.zeros(c.rows, dtype=torch.bool, device="cuda")
        none[c.starts[-1]:] = True
        for first, n in zip(c.starts, new):
            none[first + few:first + max(n, few)] = True
        check(both(tables, starts, lengths, few), none)
    # nothing is announced
    check(both(tables, starts, lengths, 0), torch.ones_like(none))


@pytest.mark.parametrize("least", [0.0, 2.0 ** -60, 2.0 ** -20])
@pytest.mark.parametrize("most", [2.0 ** 20, 2.0 ** 50, 2.0 ** 90])
def test_pages_of_tiny_values_beside_huge_ones(most, least):
    """Every fifth page holds next to nothing, the others numbers far beyond fp16: the former keep their share of the weights."""
    from energonai_b200.paged import paged_attention
    c = Case([1, 70, 5, 2], [31, 0, 200, 9], 4, 2, 64, 16, BF16, 8, seed=3)
    c.scale[1] *= most
    for page in [p for t in c.tables for p in t[::5]]:
        c.scale[1][page] = least
        if not least:
            codes = c.pool[1][page].view(torch.uint8)
            codes[codes != 0x7f] = 0
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    close(paged_attention(q, *pools, tables, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1]), *c.attention(prompt=32))


def check_values_that_are_not_finite(new, past, heads, kv_heads, dim, bits, dtype):
    """Infinities and NaN among the values: not finite is what sees them, everything else is as without them; rows whose window has left them
    behind too."""
    from energonai_b200.paged import paged_attention
    page = (16, 32, 64, 128)[(heads + len(new)) % 4]
    c = Case(new, past, heads, kv_heads, dim, page, dtype, bits, seed=heads + sum(past))
    r = torch.Generator().manual_seed(heads)
    kinds = [float("inf"), float("-inf"), float("nan")]
    bad = []                                                                # (sequence, position, key / value head, dimension, value)
    for b, (n, p) in enumerate(zip(new, past)):
        for at in {n + p - 1, p + n // 2, p + n // 3 + 1, max(0, p - 20)}:
            if at < n + p:
                bad.append((b, at, int(torch.randint(kv_heads, (1,), generator=r)), int(torch.randint(dim, (1,), generator=r)), kinds[len(bad) % 3]))
    for b, at, h, d, value in bad:
        place = (c.tables[b][at // page], h, at % page, d)
        if bits == 8:
            c.pool[1].view(torch.uint8)[place] = 0
        else:
            c.pool[1][place] = 0.0
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    for b, at, h, d, value in bad:
        place = (c.tables[b][at // page], h, at % page, d)
        if bits == 8:
            pools[1].view(torch.uint8)[place] = 0x7f if value > 0 else 0xff
        else:
            pools[1][place] = value
    group = heads // kv_heads
    for window in (0, 25, 130):
        want, tol = c.attention(window=window, prompt=64 * kv_heads // heads)
        sees = torch.zeros(c.rows, heads, dim, dtype=torch.bool)
        for b, at, h, d, _ in bad:
            for i in range(new[b]):
                pos = past[b] + i
                if at <= pos and (not window or at > pos - window):
                    sees[c.starts[b] + i, h * group:(h + 1) * group, d] = True
        sees = sees.flatten(1)
        got = paged_attention(q, *pools, tables, starts, lengths, most_new, max(c.length), window=window, k_scale=scales[0], v_scale=scales[1]).double().cpu()
        assert torch.equal(got.isfinite(), ~sees), f"window {window}: {int((got.isfinite() == sees).sum())} of {got.numel()}"
        assert bool(((got - want).abs()[~sees] <= tol[~sees]).all()), f"window {window}"


@pytest.mark.parametrize("dtype,bits", [(F16, 16), (BF16, 16), (F16, 8), (BF16, 8)])
@pytest.mark.parametrize("new,past", [([5, 3], [40, 0]), ([9, 1, 2], [250, 30, 100]), ([7], [700]), ([3, 8], [5000, 0])])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (8, 2, 128), (6, 2, 128), (7, 1, 64)])
def test_values_that_are_not_finite_reach_no_token_in_front_of_them(new, past, heads, kv_heads, dim, bits, dtype):
    check_values_that_are_not_finite(new, past, heads, kv_heads, dim, bits, dtype)



@pytest.mark.parametrize("dtype,bits", [(F16, 16), (BF16, 16), (F16, 8), (BF16, 8)])
@pytest.mark.parametrize("new,past", [([100], [0]), ([300, 70, 129], [77, 512, 0]), ([257, 1, 90], [3000, 200, 1]), ([600], [130])])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (8, 2, 128), (6, 2, 128), (7, 1, 64)])
def test_values_that_are_not_finite_reach_no_row_of_a_prompt_in_front_of_them(new, past, heads, kv_heads, dim, bits, dtype):
    from energonai_b200.gemm import device_status
    check_values_that_are_not_finite(new, past, heads, kv_heads, dim, bits, dtype)
    assert device_status()[0] == 0



@pytest.mark.parametrize("dtype,bits", [(F16, 16), (BF16, 16), (F16, 8), (BF16, 8)])
@pytest.mark.parametrize("new,past,heads,kv_heads", [([1, 80], [20000, 40], 8, 2), ([1, 3, 70], [9000, 17000, 6000], 4, 4), ([100, 1], [30000, 8400], 2, 1)])
def test_split_sequences_beside_prompts(new, past, heads, kv_heads, dtype, bits):
    """Both kernels cut keys over CTAs in one call: their partial rows share the call's scratch."""
    from energonai_b200 import _lib
    from energonai_b200.paged import paged_attention
    c = Case(new, past, heads, kv_heads, 64, 64, dtype, bits, seed=17)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    kw = dict(k_scale=scales[0], v_scale=scales[1])
    assert _lib.lib().eb_paged_attention_scratch_bytes(len(new), heads, kv_heads, 64, int(bits == 8), most_new, tables.shape[1] * 64, 0) > 0
    want, tol = c.attention(prompt=64 * kv_heads // heads)
    graph = torch.cuda.CUDAGraph()
    close(paged_attention(q, *pools, tables, starts, lengths, most_new, **kw), want, tol)
    with torch.cuda.graph(graph):
        out = paged_attention(q, *pools, tables, starts, lengths, most_new, **kw)
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(3):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                got[n].append(paged_attention(q, *pools, tables, starts, lengths, most_new, **kw))
        graph.replay()
    torch.cuda.synchronize()
    close(out, want, tol)
    assert all(torch.equal(x, out) for g in got for x in g)


def test_partial_rows_of_wide_tables():
    """Tables that address so much more than the sequences hold that the partial rows reach their bound: a CTA takes more keys then."""
    from energonai_b200 import _lib
    from energonai_b200.paged import paged_attention
    past = [30 + 7 * b for b in range(60)] + [9000, 20000, 8193, 5]
    c = Case([1] * 62 + [20, 3], past, 8, 2, 64, 16, BF16, 8, seed=23)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    need = lambda cols: _lib.lib().eb_paged_attention_scratch_bytes(64, 8, 2, 64, 1, most_new, cols * 16, 0)
    want, tol = c.attention(prompt=16)
    for cols in (tables.shape[1], 1 << 16, 1 << 20):                         # (6 MB of them, and what 256 MB hold)
        wide = torch.full((64, cols), -1, dtype=torch.int32, device="cuda")
        wide[:, :tables.shape[1]] = tables
        assert 0 < need(cols) <= 276 << 20
        close(paged_attention(q, *pools, wide, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1]), want, tol, f"{cols} columns")



def test_replay_with_other_lengths():
    """A captured step (append, attention) is replayed as sequences grow, from page to page; two captured steps share nothing."""
    from energonai_b200.paged import page_pools, paged_append, paged_attention
    B, H, G, D, page, steps = 3, 4, 2, 64, 16, 20
    past = [0, 14, 250]
    cols = 20
    c = Case([steps] * B, past, H, G, D, page, F16, 8, seed=11)
    rows = [slice(c.starts[b], c.starts[b] + steps) for b in range(B)]
    freq = frequencies(32).float().cuda()
    pools, scales = [p.cuda() for p in c.pool], [s.cuda() for s in c.scale]
    tables = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
    for b, t in enumerate(c.tables):
        tables[b, :len(t)] = torch.tensor(t, dtype=torch.int32)
    starts = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    lengths = torch.tensor(past, dtype=torch.int32, device="cuda")
    q, k, v = (torch.zeros(B, n, dtype=F16, device="cuda") for n in (H * D, G * D, G * D))
    out = torch.zeros(B, H * D, dtype=F16, device="cuda")

    def step():
        lengths.add_(1)
        turned = paged_append(q, k, v, *pools, tables, starts, lengths, 1, freq=freq, k_scale=scales[0], v_scale=scales[1])
        paged_attention(turned, *pools, tables, starts, lengths, 1, 2000, k_scale=scales[0], v_scale=scales[1], out=out)

    keep = [t.clone() for t in (*pools, *scales, lengths)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    with torch.cuda.graph(other):
        step()
    for t, old in zip((*pools, *scales, lengths), keep):
        t.copy_(old)
    got, eager = [], []
    for i in range(steps):
        for t, src in ((q, c.q), (k, c.k), (v, c.v)):
            t.copy_(torch.stack([src[r][i] for r in rows]))
        (graph if i % 3 else other).replay()
        got.append(out.clone())
    after = [t.clone() for t in (*pools, *scales)]
    for t, old in zip((*pools, *scales, lengths), keep):
        t.copy_(old)
    for i in range(steps):
        for t, src in ((q, c.q), (k, c.k), (v, c.v)):
            t.copy_(torch.stack([src[r][i] for r in rows]))
        step()
        eager.append(out.clone())
    assert all(torch.equal(a, b) for a, b in zip(got, eager))
    assert all(torch.equal(a.view(torch.uint8), t.view(torch.uint8)) for a, t in zip(after, (*pools, *scales)))
    # the last step against the restatement over what the pages hold now
    c.pool, c.scale = [p.cpu() for p in pools], [s.cpu() for s in scales]
    turned, _ = c.turned(c.q, frequencies(32).float())
    c.q = turned.flatten(1).to(F16)
    want, tol = c.attention()
    last = [r.stop - 1 for r in rows]
    close(got[-1], want[last], tol[last] + 2.0 ** -9)                        # (the queries' last bits may differ: 2^-11 of scores up to 4)


def test_refusals():
    from energonai_b200.paged import paged_append, paged_attention
    c = Case([1], [4], 4, 2, 64, 16, F16, 8, seed=1)
    (q, k, v), pools, scales, (tables, starts, lengths, most_new) = c.device()
    kw = dict(k_scale=scales[0], v_scale=scales[1])
    for fn, args in ((paged_append, (q, k, v)), (paged_attention, (q,))):
        for bad, words in ((dict(k_scale=None), "scales"), (dict(k_scale=None, v_scale=None), "pools of"), (dict(k_scale=scales[0].half()), "scales")):
            with pytest.raises(RuntimeError, match=words):
                fn(*args, *pools, tables, starts, lengths, most_new, **{**kw, **bad})
        for bad in ((tables.long(), starts, lengths), (tables, starts[:1], lengths), (tables, starts, lengths[:0]), (tables[0], starts, lengths)):
            with pytest.raises(RuntimeError, match="int32"):
                fn(*args, *pools, *bad, most_new, **kw)
        with pytest.raises(RuntimeError, match="pools"):
            fn(*args, pools[0], pools[1][:1], tables, starts, lengths, most_new, **kw)
        with pytest.raises(RuntimeError, match="CUDA"):
            fn(*args, pools[0], pools[1], tables.cpu(), starts, lengths, most_new, **kw)
    with pytest.raises(RuntimeError, match="contiguous columns"):
        paged_append(q, k.bfloat16(), v, *pools, tables, starts, lengths, most_new, **kw)
    with pytest.raises(RuntimeError, match="frequencies"):
        paged_append(q, k, v, *pools, tables, starts, lengths, most_new, freq=torch.ones(33, device="cuda"), **kw)
    with pytest.raises(RuntimeError, match="unsupported dtype|fp16"):
        paged_attention(q.float(), pools[0].float(), pools[1].float(), tables, starts, lengths, most_new)
    with pytest.raises(RuntimeError, match="window"):
        paged_attention(q, *pools, tables, starts, lengths, most_new, window=-1, **kw)
