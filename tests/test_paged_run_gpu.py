"""An attention layer as a server of many requests runs it: projections with an adapter per request, new tokens into paged caches, attention over
them, the output projection; prompts, single tokens, and both in one batch.  Every stage is held to its restatement in 64 bits on
what the stage before left."""
import pytest
import torch

from paged_plain import Case
from test_adapter_gpu import UNIT, Case as Adapters
from test_paged_gpu import check_append, close, frequencies

pytestmark = pytest.mark.gpu


def product(x, c, w):
    """(x w^T + adapters, tolerance), as in the adapters' own test."""
    y, size = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    c.x = x
    delta, tol = c.delta()
    return y + delta, UNIT[c.dtype] * (y + delta).abs() + tol + (2.0 ** -23 * x.shape[1] / 16 + 2.0 ** -20) * size


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 16])
def test_an_attention_layer_serves_many_requests(bits, dtype):
    from energonai_b200.adapter import adapter_product
    from energonai_b200.gemm import device_status
    from energonai_b200.paged import page_pools, paged_append, paged_attention, paged_batch
    H, G, D, page, width, pages = 8, 2, 64, 16, 512, 64
    B, columns = 4, (H + 2 * G) * D
    into, out_of = Adapters([1], width, columns, 16, 3, dtype, seed=1), Adapters([1], H * D, width, 16, 3, dtype, seed=2)
    freq = frequencies(D // 2).float()
    pools = page_pools(pages, page, G, D, torch.float8_e4m3fn if bits == 8 else dtype)
    k_pages, v_pages, k_scale, v_scale = pools
    for p in (k_pages, v_pages):
        p.view(torch.uint8).fill_(0x7f)                                       # NaN, or close to it, wherever nothing was written
    g = torch.Generator().manual_seed(5)
    free = torch.randperm(pages, generator=g).tolist()
    tables, length = [[] for _ in range(B)], [0] * B
    index = torch.tensor([2, -1, 0, 2], dtype=torch.int32)
    for new in ([70, 5, 0, 33], [1, 1, 1, 1], [1, 90, 1, 0], [3, 1, 2, 1], [1, 1, 1, 1]):
        for b in range(B):
            length[b] += new[b]
            while len(tables[b]) * page < length[b]:
                tables[b].append(free.pop())
        t, starts, lengths, most_new, most_length = paged_batch(new, length, tables, pages, page)
        rows = sum(new)
        x = torch.randn(rows, width, generator=g).to(dtype)
        common = (index.cuda(), starts, most_new)
        proj = adapter_product(x.cuda(), into.w.cuda(), into.a.cuda(), into.b.cuda(), into.scales.cuda(), *common)
        for c in (into, out_of):
            c.new, c.starts, c.rows, c.index = new, starts.tolist(), rows, index
        close(proj, *product(x, into, into.w), "projection")

        q, k, v = proj[:, :H * D], proj[:, H * D:(H + G) * D], proj[:, (H + G) * D:]
        c = Case([0], [0], H, G, D, page, dtype, bits)
        c.new, c.length, c.past, c.tables, c.starts, c.rows, c.pages = new, list(length), [n - m for n, m in zip(length, new)], tables, starts.tolist(), rows, pages
        c.q, c.k, c.v = (y.cpu() for y in (q, k, v))
        c.pool, c.scale = [p.cpu() for p in pools[:2]], [s.cpu() if s is not None else None for s in pools[2:]]
        turned = paged_append(q, k, v, k_pages, v_pages, t, starts, lengths, most_new, freq=freq.cuda(), k_scale=k_scale, v_scale=v_scale)
        check_append(c, D // 2, turned, pools[:2], pools[2:])

        c.q, c.pool, c.scale = turned.cpu(), [p.cpu() for p in pools[:2]], [s.cpu() if s is not None else None for s in pools[2:]]
        attended = paged_attention(turned, k_pages, v_pages, t, starts, lengths, most_new, most_length, k_scale=k_scale, v_scale=v_scale)
        close(attended, *c.attention(prompt=64 * G // H), "attention")

        y = adapter_product(attended, out_of.w.cuda(), out_of.a.cuda(), out_of.b.cuda(), out_of.scales.cuda(), *common)
        close(y, *product(attended.cpu(), out_of, out_of.w), "output")
    assert device_status()[0] == 0


def test_two_streams_at_once():
    """Calls on two streams share no scratch."""
    from energonai_b200.adapter import adapter_product
    from energonai_b200.paged import paged_attention
    cases = [Case([1, 1], [9000, 5000], 8, 2, 64, 16, torch.float16, 8, seed=s) for s in (1, 2)]
    more = [Adapters([40, 3], 512, 256, 16, 2, torch.float16, seed=s) for s in (3, 4)]

    def run(c, a):
        (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c
        x, w, rest = a
        return paged_attention(q, *pools, tables, starts, lengths, most_new, k_scale=scales[0], v_scale=scales[1]), adapter_product(x, w, *rest)

    inputs = [(c.device(), (a.x.cuda(), a.w.cuda(), a.device())) for c, a in zip(cases, more)]
    want = [run(*i) for i in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                got[n].append(run(*inputs[n])[0])
    torch.cuda.synchronize()
    for n in (0, 1):
        assert all(torch.equal(o, want[n][0]) for o in got[n])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,width,columns", [([1] * 16, 5120, 5120), ([5, 27], 2048, 8192), ([2], 4096, 12288), ([40, 3], 512, 256), ([1] * 9, 512, 256)])
def test_adapters_on_two_streams(new, width, columns, dtype):
    """Products of few rows of a large weight are split over K and meet in scratch: eager calls on two streams, and two captured graphs that are
    replayed on two streams, get the bits that they get alone."""
    from energonai_b200.adapter import adapter_product
    from energonai_b200.gemm import device_status
    cases = [Adapters(new, width, columns, 16, 2, dtype, seed=s) for s in (3, 4)]
    inputs = [(c.x.cuda(), c.w.cuda(), *c.device()) for c in cases]
    want = [adapter_product(*i) for i in inputs]
    close(want[0], *product(cases[0].x, cases[0], cases[0].w))
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for n in (0, 1):
        with torch.cuda.graph(graphs[n]):
            outs.append([adapter_product(*inputs[n]) for _ in range(8)])
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                got[n].append(adapter_product(*inputs[n]))
    torch.cuda.synchronize()
    for n in (0, 1):
        assert all(torch.equal(y, want[n]) for y in got[n])
    for _ in range(5):
        for n in (0, 1):
            with torch.cuda.stream(streams[n]):
                graphs[n].replay()
        torch.cuda.synchronize()
        for n in (0, 1):
            assert all(torch.equal(y, want[n]) for y in outs[n])
            for y in outs[n]:
                y.fill_(5.0)
        torch.cuda.synchronize()
    assert device_status()[0] == 0


def test_tables_of_a_wider_table():
    from energonai_b200.paged import paged_attention
    c = Case([1, 7], [40, 90], 4, 2, 64, 32, torch.bfloat16, 16, seed=7)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    wide = torch.full((2, 50), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + tables.shape[1]] = tables
    part = wide[:, 3:3 + tables.shape[1]]
    got = paged_attention(q, *pools, part, starts, lengths, most_new)
    assert torch.equal(got, paged_attention(q, *pools, tables, starts, lengths, most_new))
    close(got, *c.attention())


@pytest.mark.parametrize("dtype,bits", [(torch.float16, 16), (torch.bfloat16, 8)])
def test_long_sequences_among_many(bits, dtype):
    """So many sequences that none is split: hundreds of tiles per warp, and one sequence that is long enough to be split all the same."""
    from energonai_b200.paged import paged_attention
    past = [4000, 2047, 2100, 9000, 5] + [40 + b for b in range(43)]
    c = Case([1] * 48, past, 8, 8, 64, 16, dtype, bits, seed=13)
    (q, _, _), pools, scales, (tables, starts, lengths, most_new) = c.device()
    for window in (0, 3000):
        got = paged_attention(q, *pools, tables, starts, lengths, most_new, window=window, k_scale=scales[0], v_scale=scales[1])
        close(got, *c.attention(window=window))


@pytest.mark.parametrize("bits", [8, 16])
def test_replayed_batches_of_prompts_and_steps(bits):
    """One captured call serves other batches: who brings a prompt, who a token, how long all are."""
    from energonai_b200.paged import paged_append, paged_attention
    H, G, D, page, rows, cols = 8, 2, 128, 32, 200, 40
    first = Case([100, 1, 99], [0, 30, 5], H, G, D, page, torch.float16, bits, seed=31)
    (q, k, v), pools, scales, (_, starts, lengths, _) = first.device()
    pages = 100
    big = [torch.zeros((pages,) + p.shape[1:], dtype=p.dtype, device="cuda") for p in pools]
    zs = [torch.ones(pages, G, device="cuda") if s is not None else None for s in scales]
    tables = torch.full((3, cols), -1, dtype=torch.int32, device="cuda")
    freq = frequencies(64).float().cuda()
    out = torch.zeros_like(q)

    def call():
        turned = paged_append(q, k, v, *big, tables, starts, lengths, 150, freq=freq, k_scale=zs[0], v_scale=zs[1])
        paged_attention(turned, *big, tables, starts, lengths, 150, 1200, k_scale=zs[0], v_scale=zs[1], out=out)
        return turned

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed, (new, past) in enumerate((([100, 1, 99], [0, 30, 5]), ([1, 150, 1], [700, 0, 1000]), ([1, 1, 1], [5, 6, 900]), ([0, 20, 120], [3, 200, 64]))):
        c = Case(new, past, H, G, D, page, torch.float16, bits, seed=40 + seed, pad_rows=rows - sum(new))
        (q1, k1, v1), p1, s1, (t1, st, le, _) = c.device()
        for to, src in ((q, q1), (k, k1), (v, v1), (starts, st), (lengths, le)):
            to.copy_(src)
        for to, src in zip(big, p1):
            to.view(torch.uint8)[:c.pages].copy_(src.view(torch.uint8))
        for to, src in zip(zs, s1):
            if src is not None:
                to[:c.pages].copy_(src)
        tables.fill_(-1)
        tables[:, :t1.shape[1]] = t1
        keep = [t.clone() for t in (*big, *(z for z in zs if z is not None))]
        out.fill_(7.0)
        graph.replay()
        got = out.clone()
        after = [t.clone() for t in (*big, *(z for z in zs if z is not None))]
        for t, old in zip((*big, *(z for z in zs if z is not None)), keep):
            t.copy_(old)
        out.fill_(7.0)
        turned = call()
        assert torch.equal(got, out) and all(torch.equal(a.view(torch.uint8), t.view(torch.uint8)) for a, t in zip(after, (*big, *(z for z in zs if z is not None))))
        assert bool((got[sum(new):] == 7.0).all())
        # against the restatement, over the pages and the turned queries that the call left
        c.q, c.pool, c.scale = turned.cpu(), [b[:c.pages].cpu() for b in big], [z[:c.pages].cpu() if z is not None else None for z in zs]
        want, tol = c.attention(prompt=16)
        close(got[:sum(new)], want[:sum(new)], tol[:sum(new)])


def test_pools_beyond_32_bit_offsets():
    """Pages behind 2^31 elements and 2^32 bytes: the same bits as from the front of the pool."""
    from energonai_b200.paged import paged_append, paged_attention
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 20 GB")
    for bits, dtype in ((16, torch.float16), (8, torch.bfloat16)):
        c = Case([1, 90, 2], [300, 40, 9], 8, 8, 128, 128, dtype, bits, seed=51)
        (q, k, v), pools, scales, (tables, starts, lengths, most_new) = c.device()
        per_page = 8 * 128 * 128
        pages = (1 << (31 if bits == 16 else 32)) // per_page + 16 + c.pages
        shift = pages - c.pages
        far = [torch.empty((pages, 8, 128, 128), dtype=p.dtype, device="cuda") for p in pools]
        zs = [torch.ones((pages, 8), device="cuda") if s is not None else None for s in scales]
        for to, src in zip(far, pools):
            to[shift:].view(torch.uint8).copy_(src.view(torch.uint8))
        for to, src in zip(zs, scales):
            if src is not None:
                to[shift:] = src
        moved = torch.where(tables >= 0, tables + shift, tables)
        freq = frequencies(64).float().cuda()
        results = []
        for p, z, t in ((pools, scales, tables), (far, zs, moved)):
            turned = paged_append(q, k, v, *p, t, starts, lengths, most_new, freq=freq, k_scale=z[0], v_scale=z[1])
            results.append(paged_attention(turned, *p, t, starts, lengths, most_new, k_scale=z[0], v_scale=z[1]))
        assert torch.isfinite(results[0]).all() and torch.equal(*results)
        assert all(torch.equal(a[shift:].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(far, pools))
        del far
        torch.cuda.empty_cache()
