"""Low-rank adapters of many requests against products in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


class Case:
    def __init__(self, new, width, columns, rank, adapters, dtype, seed=0, pad_rows=0):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *shape: torch.randn(*shape, generator=g)
        self.new, self.starts = new, [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.rows, self.dtype, self.most_new = self.starts[-1] + pad_rows, dtype, max(1, max(new))
        self.x, self.w = rnd(self.rows, width).to(dtype), (rnd(columns, width) / width ** 0.5).to(dtype)
        self.a, self.b = (rnd(adapters, rank, width) / width ** 0.5).to(dtype), (rnd(adapters, columns, rank) / rank ** 0.5).to(dtype)
        self.bias, self.scales = rnd(columns).to(dtype), 0.25 + torch.rand(adapters, generator=g)
        self.index = torch.randint(-1, adapters, (len(new),), generator=g, dtype=torch.int32)
        self.index[-1] = 0

    def device(self):
        return [t.cuda() for t in (self.a, self.b, self.scales, self.index)] + [torch.tensor(self.starts, dtype=torch.int32, device="cuda"), self.most_new]

    def delta(self):
        """(delta, tolerance): its rounding, and fp32 sums of `width` products: a tile adds up 16 products and rounds (truncates) into the
        accumulator once, 2^-23 of the running sum per tile of a slice of 1 / 4 or less of the width, bounded by
        2^-23 width / 64 + 2^-20 of the sum of magnitudes; the second product adds 2^-20, and the pieces of the low-rank row 2^-16 (bf16)."""
        out, size = torch.zeros(self.rows, self.b.shape[1], dtype=torch.float64), torch.zeros(self.rows, self.b.shape[1], dtype=torch.float64)
        for s, i in enumerate(self.index.tolist()):
            if 0 <= i < self.a.shape[0] and self.new[s]:
                r = slice(self.starts[s], self.starts[s + 1])
                x, a, b, scale = self.x[r].double(), self.a[i].double(), self.b[i].double(), float(self.scales[i])
                out[r] = scale * (x @ a.T) @ b.T
                size[r] = scale * (x.abs() @ a.abs().T) @ b.abs().T
                if self.dtype == BF16:
                    size[r] += scale * 2.0 ** 4 * (x @ a.T).abs() @ b.abs().T                # (2^-16, in units of 2^-20)
        return out, UNIT[self.dtype] * out.abs() + (2.0 ** -23 * self.x.shape[1] / 64 + 2.0 ** -19) * size


def close(got, want, tol):
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert float(((got - want).abs() - tol).max()) <= 0


SHAPES = [([1], 64, 64, 8, 1), ([1] * 9, 768, 2304, 16, 4), ([1] * 70, 5120, 1024, 24, 90), ([5, 1, 40, 0, 2], 200, 136, 32, 3), ([130, 17, 64], 1024, 520, 64, 2),
          ([33], 136, 1032, 128, 2), ([16, 16], 4096, 264, 8, 2), ([15, 1, 1], 2048, 40, 120, 5)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,width,columns,rank,adapters", SHAPES)
def test_delta_and_product(new, width, columns, rank, adapters, dtype):
    from energonai_b200.adapter import adapter_delta, adapter_product
    c = Case(new, width, columns, rank, adapters, dtype, seed=width + rank, pad_rows=3)
    want, tol = c.delta()
    close(adapter_delta(c.x.cuda(), *c.device()), want, tol)
    y = c.x.double() @ c.w.double().T + c.bias.double()
    size = c.x.double().abs() @ c.w.double().abs().T + c.bias.double().abs()
    got = adapter_product(c.x.cuda(), c.w.cuda(), *c.device(), bias=c.bias.cuda())
    # the sum is rounded once, delta before it
    close(got, y + want, UNIT[dtype] * (y + want).abs() + tol + (2.0 ** -23 * width / 16 + 2.0 ** -20) * size)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("x,a,b", [(2.0 ** 9, 2.0 ** 6, 2.0 ** -6), (2.0 ** -8, 2.0 ** -6, 2.0 ** 6)])
@pytest.mark.parametrize("new,rank", [([1, 3, 16], 8), ([5, 9], 40), ([70, 1], 16), ([33], 24), ([40, 100], 64), ([64], 120)])
def test_low_rank_rows_beyond_half_precision(new, rank, x, a, b, dtype):
    """The low-rank row itself may be larger or smaller than fp16 can say; the result is not."""
    from energonai_b200.adapter import adapter_delta
    c = Case(new, 512, 264, rank, 2, dtype, seed=rank, pad_rows=2)
    c.x, c.a, c.b = c.x * x, c.a * a, c.b * b
    close(adapter_delta(c.x.cuda(), *c.device()), *c.delta())


def test_many_rows_behind_the_last_sequence():
    from energonai_b200.adapter import adapter_delta
    c = Case([1, 2], 64, 96, 8, 2, F16, seed=3, pad_rows=500)
    delta = adapter_delta(c.x.cuda(), *c.device())
    close(delta, *c.delta())
    assert not delta[3:].any()


@pytest.mark.parametrize("most_new", [16, 64])
def test_rows_that_were_not_announced_get_nothing(most_new):
    from energonai_b200.adapter import adapter_delta
    c = Case([200, 3], 64, 96, 8, 2, BF16, seed=6)
    c.index[:] = 1
    want, tol = c.delta()
    c.most_new = most_new
    got = adapter_delta(c.x.cuda(), *c.device())
    assert not got[most_new:200].any()
    want[most_new:200] = 0
    close(got, want, tol)


@pytest.mark.parametrize("most_new", [6, 40])
def test_rows_in_front_of_the_first_sequence(most_new):
    """A part of a batch: the later sequences' starts and adapters alone."""
    from energonai_b200.adapter import adapter_delta
    c = Case([30, 5, 6], 64, 96, 8, 2, BF16, seed=7, pad_rows=2)
    c.index[:] = 1
    a, b, scales, index, starts, _ = c.device()
    torch.full((43, 96), 5.0, dtype=BF16, device="cuda")                     # (what an output that is not written would hold)
    got = adapter_delta(c.x.cuda(), a, b, scales, index[1:], starts[1:], most_new)
    want, tol = c.delta()
    want[:30] = 0
    close(got, want, tol)
    assert not got[:30].any()
    assert not adapter_delta(c.x.cuda(), a, b, scales, index[:1], starts[:1].expand(2).contiguous(), 0).any()


def test_other_indices_are_none():
    from energonai_b200.adapter import adapter_delta
    c = Case([2, 3, 1], 64, 96, 8, 2, BF16, seed=4)
    c.index = torch.tensor([2, -7, 1 << 30], dtype=torch.int32)
    assert not adapter_delta(c.x.cuda(), *c.device()).any()


def test_strided_rows_and_output():
    from energonai_b200.adapter import adapter_product
    c = Case([4, 30], 256, 128, 16, 2, F16, seed=5)
    wide, out = torch.zeros(34, 512, dtype=F16, device="cuda"), torch.zeros(34, 384, dtype=F16, device="cuda")
    wide[:, 128:384] = c.x.cuda()
    got = adapter_product(wide[:, 128:384], c.w.cuda(), *c.device(), out=out[:, 128:256])
    assert torch.equal(got, adapter_product(c.x.cuda(), c.w.cuda(), *c.device()))
    assert not out[:, :128].any() and not out[:, 256:].any()


def test_replay_with_other_adapters():
    from energonai_b200.adapter import adapter_product
    c = Case([1] * 6, 512, 256, 16, 4, BF16, seed=6)
    x, w, rest = c.x.cuda(), c.w.cuda(), c.device()
    adapter_product(x, w, *rest)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = adapter_product(x, w, *rest)
    for seed in range(3):
        other = Case([1] * 6, 512, 256, 16, 4, BF16, seed=20 + seed)
        x.copy_(other.x)
        rest[3].copy_(other.index)
        graph.replay()
        assert torch.equal(y, adapter_product(x, w, *rest))


def test_refusals():
    from energonai_b200.adapter import adapter_delta, adapter_product
    c = Case([1, 2], 64, 96, 8, 2, F16, seed=1)
    x, w, (a, b, scales, index, starts, most_new) = c.x.cuda(), c.w.cuda(), c.device()
    for bad, words in (((a[:, :, :32], b, scales, index, starts), "required"), ((a.bfloat16(), b, scales, index, starts), "type of x"), ((a, b, scales.half(), index, starts), "fp32 scale"),
                       ((a, b, scales, index.long(), starts), "int32"), ((a, b, scales, index, starts[:2]), "int32"), ((a, b[:1], scales, index, starts), "required")):
        with pytest.raises(RuntimeError, match=words):
            adapter_delta(x, *bad, most_new)
    with pytest.raises(RuntimeError, match="rank 4"):
        adapter_delta(x, a[:, :4].contiguous(), b[:, :, :4].contiguous(), scales, index, starts, most_new)
    with pytest.raises(RuntimeError, match="shared weight"):
        adapter_product(x, w[:8], a, b, scales, index, starts, most_new)
    with pytest.raises(RuntimeError, match="bias"):
        adapter_product(x, w, a, b, scales, index, starts, most_new, bias=torch.zeros(96, device="cuda"))


def same_kind(got, want, tol):
    """Infinities with their sign and NaN where they belong, the rest within the tolerance."""
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    there = want.isfinite()
    assert bool(((got - want).abs()[there] <= tol[there]).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,rank", [([1, 3, 16], 8), ([5, 9], 40), ([70, 1], 16), ([40, 100], 64), ([64], 120)])
def test_infinities_of_low_rank_rows(new, rank, dtype):
    """An infinity keeps its sign, NaN stays NaN."""
    from energonai_b200.adapter import adapter_delta
    c = Case(new, 264, 136, rank, 2, dtype, seed=rank + len(new), pad_rows=2)
    c.index[:] = 1
    c.x[:, 7] = 0.0
    c.x[0, 7], c.x[c.rows - 3, 7] = 1.0, -2.0                                # (the rows that meet them; for the others 0 * infinity is NaN)
    rows = [0, c.rows - 3]
    for value in (float("inf"), float("-inf"), float("nan")):
        c.a[1, rank - 3, 7] = value
        want, tol = c.delta()
        same_kind(adapter_delta(c.x.cuda(), *c.device())[rows], want[rows], tol[rows])


def test_low_rank_values_at_the_end_of_the_range():
    """A low-rank value between bf16's and fp32's largest; and fp16's scaled far beyond its own range."""
    from energonai_b200.adapter import adapter_delta
    for dtype, x, a, b, scale in ((BF16, (1.0, 1.0), (torch.finfo(BF16).max, 1.5 * 2.0 ** 119), 2.0 ** -30, 1.0), (F16, (2.0 ** 14, 2.0 ** 14), (2.0 ** 13, 2.0 ** 12), 2.0 ** -20, 2.0 ** 97)):
        for new in (3, 70):
            c = Case([new], 64, 64, 16, 1, dtype, seed=2)
            c.x.zero_()
            c.a.zero_()
            c.x[:, 0], c.x[:, 1] = x
            c.a[0, 3, 0], c.a[0, 3, 1] = a
            c.b[:] = b
            c.scales[:] = scale
            want, tol = c.delta()
            if dtype == F16:                                                 # (beyond fp16 in the end: infinite, not NaN)
                assert bool((adapter_delta(c.x.cuda(), *c.device()) == float("inf")).all())
                c.b *= -1.0
                assert bool((adapter_delta(c.x.cuda(), *c.device()) == float("-inf")).all())
            else:
                close(adapter_delta(c.x.cuda(), *c.device()), want, tol)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("most_new", [1, 10, 15, 17, 63, 65, 70])
def test_the_adapter_ends_at_the_announced_rows(most_new, dtype):
    from energonai_b200.adapter import adapter_delta, adapter_product
    c = Case([100, 12, 30], 136, 264, 24, 2, dtype, seed=most_new, pad_rows=1)
    c.index[:] = torch.tensor([1, -1, 0], dtype=torch.int32)
    want, tol = c.delta()
    c.most_new = most_new
    for first, n in ((0, 100), (112, 30)):
        want[first + most_new:first + n], tol[first + most_new:first + n] = 0, 0
    close(adapter_delta(c.x.cuda(), *c.device()), want, tol)
    y = c.x.double() @ c.w.double().T
    size = c.x.double().abs() @ c.w.double().abs().T
    close(adapter_product(c.x.cuda(), c.w.cuda(), *c.device()), y + want, UNIT[dtype] * (y + want).abs() + tol + (2.0 ** -23 * 136 / 16 + 2.0 ** -20) * size)


@pytest.mark.parametrize("new", [[3, 1], [40], [70, 30, 1]])
def test_an_adapters_part_beyond_half_precision(new):
    """The adapter's part alone is more than fp16 holds, its sum with the shared projection is not."""
    from energonai_b200.adapter import adapter_product
    c = Case(new, 256, 136, 16, 2, F16, seed=len(new), pad_rows=2)
    c.index[:] = 0
    c.index[-1] = 1
    # x W^T near -100,000, the adapters' part near 100,000: one column of ones carries both
    c.x[:, 0] = 256.0
    c.w[:, 0] = -390.0
    c.a[:, :, 0] = 0.0
    c.a[:, 0, 0] = 4.0
    c.b[:, :, 0] = 97.5
    c.scales[:] = 1.0
    want, tol = c.delta()
    y = c.x.double() @ c.w.double().T
    size = c.x.double().abs() @ c.w.double().abs().T
    n = sum(new)
    assert float(want[:n].abs().min()) > 65504 and float((y + want)[:n].abs().max()) < 30000
    got = adapter_product(c.x.cuda(), c.w.cuda(), *c.device())
    tol = tol - UNIT[F16] * want.abs() + UNIT[F16] * (y + want).abs() + (2.0 ** -23 * 256 / 16 + 2.0 ** -20) * size
    close(got[:n], (y + want)[:n], tol[:n])
    assert bool((got[n:].double().cpu() == float("-inf")).all())             # (rows of no sequence: the shared projection alone, beyond fp16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new", [[4, 30], [1]])
def test_output_rows_of_any_stride(new, dtype):
    from energonai_b200.adapter import adapter_product
    c = Case(new, 256, 128, 16, 2, dtype, seed=5)
    wide = torch.zeros(c.rows, 132, dtype=dtype, device="cuda")
    got = adapter_product(c.x.cuda(), c.w.cuda(), *c.device(), out=wide[:, :128])
    assert got.data_ptr() == wide.data_ptr() and not wide[:, 128:].any()
    want, tol = c.delta()
    y, size = c.x.double() @ c.w.double().T, c.x.double().abs() @ c.w.double().abs().T
    close(got, y + want, UNIT[dtype] * (y + want).abs() + tol + (2.0 ** -23 * 256 / 16 + 2.0 ** -20) * size)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new", [[3, 1], [60, 20]])
def test_the_shared_projection_of_a_padded_batch(new, dtype):
    """Many rows in front of the first sequence and behind the last: x W^T + bias there, rounded once."""
    from energonai_b200.adapter import adapter_delta, adapter_product
    c = Case([300] + new, 128, 520, 16, 2, dtype, seed=8, pad_rows=700)
    c.index[:] = 1
    a, b, scales, index, starts, _ = c.device()
    some = (a, b, scales, index[1:], starts[1:], max(new))
    want, tol = c.delta()
    want[:300], tol[:300] = 0, 0
    delta = adapter_delta(c.x.cuda(), *some)
    close(delta, want, tol)
    assert not delta[:300].any() and not delta[c.starts[-1]:].any()
    y = c.x.double() @ c.w.double().T + c.bias.double()
    size = c.x.double().abs() @ c.w.double().abs().T + c.bias.double().abs()
    got = adapter_product(c.x.cuda(), c.w.cuda(), *some, bias=c.bias.cuda())
    close(got, y + want, UNIT[dtype] * (y + want).abs() + tol + (2.0 ** -23 * 128 / 16 + 2.0 ** -20) * size)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_nothing_is_announced(dtype):
    from energonai_b200.adapter import adapter_delta, adapter_product
    c = Case([5, 2], 128, 264, 16, 2, dtype, seed=3, pad_rows=1)
    c.index[:] = 1
    c.most_new = 0
    assert not adapter_delta(c.x.cuda(), *c.device()).any()
    y, size = c.x.double() @ c.w.double().T, c.x.double().abs() @ c.w.double().abs().T
    out = torch.full((c.rows, 264), 3.0, dtype=dtype, device="cuda")
    for given in (None, out):
        got = adapter_product(c.x.cuda(), c.w.cuda(), *c.device(), out=given)
        close(got, y, UNIT[dtype] * y.abs() + (2.0 ** -23 * 128 / 16 + 2.0 ** -20) * size)
    assert got.data_ptr() == out.data_ptr()
