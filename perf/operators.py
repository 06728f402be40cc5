"""Cases of serving many requests at once out of a paged cache.  A packed batch: rows starts[b] to starts[b + 1] are the
new tokens of sequence b, lengths[b] its positions in the cache with the new ones, tables[b] the pages that hold them.

  append     keys and values of new tokens go to their pages, with the position rotation of queries and keys on the way;
             pages in the model's type or in 8 bits (e4m3) with a scale for each page and head
  attention  the new tokens' causal attention over those pages: single tokens, a few, prompt chunks behind a cached past
  adapter    a projection with a low-rank adapter per request beside the shared weight

Lengths follow from the case, values from the seed."""
import math
import random

import torch

own = False
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


# ---- the cases ----------------------------------------------------------------------------------------------
def listed():
    return [
        # generation step of a served batch on 8-bit pages, odd lengths: one token per sequence
        dict(name="append_step", kind="append", batch=64, heads=32, kv_heads=8, dim=128, new=1, past=3000, page=16, bits=8, pairs=64, dtype="bf16"),
        # prompts and prompt chunks of odd lengths into 8-bit pages, behind pasts that end inside a page
        dict(name="append_prompts", kind="append", batch=9, heads=32, kv_heads=8, dim=128, new=1500, past=700, page=32, bits=8, pairs=64, dtype="bf16"),
        # prompts of a model with learned positions: nothing to rotate, 16-bit pages
        dict(name="append_13b", kind="append", batch=5, heads=40, kv_heads=40, dim=128, new=1100, past=0, page=64, bits=16, pairs=0, dtype="fp16"),
        # one user's chat with a small model: almost no work
        dict(name="step_small", kind="attention", batch=1, heads=12, kv_heads=12, dim=64, new=1, past=36, page=16, bits=16, window=0, dtype="fp16"),
        # the headline model's generation step at its benchmark's batch and length
        dict(name="step_13b", kind="attention", batch=16, heads=40, kv_heads=40, dim=128, new=1, past=640, page=64, bits=16, window=0, dtype="fp16"),
        # a served batch of ragged lengths on 8-bit pages, heads in groups
        dict(name="step_batch", kind="attention", batch=64, heads=32, kv_heads=8, dim=128, new=1, past=4095, page=16, bits=8, window=0, dtype="bf16"),
        # one request over a very long document
        dict(name="step_long", kind="attention", batch=1, heads=32, kv_heads=8, dim=128, new=1, past=131000, page=64, bits=8, window=0, dtype="bf16"),
        # a few draft tokens per sequence, checked at once; a sliding window
        dict(name="drafts", kind="attention", batch=24, heads=16, kv_heads=4, dim=128, new=5, past=2500, page=32, bits=16, window=1024, dtype="bf16"),
        # prompt chunks behind a long cached past in 8 bits
        dict(name="chunks", kind="attention", batch=3, heads=32, kv_heads=8, dim=128, new=1024, past=7000, page=64, bits=8, window=0, dtype="bf16"),
        # whole prompts of odd lengths, first pass, 16-bit pages
        dict(name="prompts", kind="attention", batch=6, heads=40, kv_heads=40, dim=128, new=1531, past=0, page=16, bits=16, window=0, dtype="fp16"),
        # generation step: every request with an adapter of its own
        dict(name="adapter_step", kind="adapter", batch=48, new=1, width=5120, columns=5120, rank=16, adapters=64, bias=True, dtype="fp16"),
        # prompts of odd lengths, one request without an adapter
        dict(name="adapter_prompts", kind="adapter", batch=6, new=900, width=4096, columns=6144, rank=64, adapters=8, bias=False, dtype="bf16"),
    ]


def spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(12, 12, 64), (16, 16, 64), (16, 4, 128), (32, 8, 128), (40, 40, 128), (56, 56, 128)]


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "adapter"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "adapter":
        width, columns = rng.choice([(768, 2304), (1024, 1024), (2048, 2560), (4096, 6144), (5120, 5120)])
        step = rng.random() < 0.5
        batch = spread(rng, 1, 128 if step else 12)
        return dict(kind=kind, batch=batch, new=1 if step else spread(rng, 2, 4000 // batch), width=width, columns=columns, rank=8 * rng.choice([1, 2, 2, 3, 4, 8, 16]),
                    adapters=spread(rng, 1, 64), bias=rng.random() < 0.5, dtype=dtype)
    heads, kv_heads, dim = rng.choice(HEADS)
    common = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]), bits=rng.choice([8, 16]), dtype=dtype)
    if kind == "append":
        step = rng.random() < 0.4
        batch = spread(rng, 1, 128 if step else 12)
        return dict(common, batch=batch, new=1 if step else spread(rng, 2, 4000 // batch), past=spread(rng, 1, 4000), pairs=rng.choice([0, dim // 4, dim // 2, dim // 2]))
    form = rng.choice(["step", "step", "few", "chunk"])
    window = rng.choice([0, 0, spread(rng, 16, 4096)])
    if form == "chunk":
        new, past = spread(rng, 17, 1200), spread(rng, 1, 5000)
        most = round(2e11 / (4 * heads * dim * new * (new + past)))
        return dict(common, batch=spread(rng, 1, max(1, min(12, most))), new=new, past=past, window=window)
    most = 750_000 // kv_heads                                          # positions of the batch
    past = spread(rng, 1, min(most, 130000))
    return dict(common, batch=spread(rng, 1, min(128, most // past)), new=1 if form == "step" else rng.randint(2, 16), past=past, window=window)


def lengths(case):
    """(new tokens, positions) of each sequence, on the host: the first has the case's sizes in full, the others from half of them on."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    ragged = lambda n: rng.randint((n + 1) // 2, n) if n > 1 else n
    new = [case["new"]] + [ragged(case["new"]) for _ in range(case["batch"] - 1)]
    past = [case.get("past", 0)] + [ragged(case.get("past", 0)) for _ in range(case["batch"] - 1)]
    return new, [n + p for n, p in zip(new, past)]


# ---- inputs -------------------------------------------------------------------------------------------------
def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def eight_bit(x):
    """x [..., rows, dim] -> codes and a scale for each block of rows, a power of two."""
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((-2, -1)) / 448)))
    return (x / scale[..., None, None]).to(E4M3), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    new, length = lengths(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows, batch = starts[-1], case["batch"]
    state = dict(case=case, starts=ints(starts), most_new=max(new))
    if case["kind"] == "adapter":
        width, columns, rank, count = case["width"], case["columns"], case["rank"], case["adapters"]
        index = torch.randint(0, count, (batch,), generator=g, device="cuda", dtype=torch.int32) if count < batch else torch.randperm(
            count, generator=g, device="cuda")[:batch].to(torch.int32)
        if batch > 2:
            index[batch // 2] = -1
        return dict(state, x=randn(rows, width).to(dtype), w=(randn(columns, width) / width ** 0.5).to(dtype),
                    a=(randn(count, rank, width) / width ** 0.5).to(dtype), b=(randn(count, columns, rank) / rank ** 0.5).to(dtype),
                    scales=0.25 + 0.5 * torch.rand(count, generator=g, device="cuda"), index=index,
                    bias=randn(columns).to(dtype) if case["bias"] else None)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    need = [-(-n // page) for n in length]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)              # pages lie in no order
    tables = torch.zeros((batch, max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    state.update(tables=tables, lengths=ints(length), most_length=max(length))
    size = torch.exp2(torch.randint(-2, 3, (2, pages, kv_heads, 1, 1), generator=g, device="cuda").float() / 2)   # blocks differ in magnitude
    for name, z in (("k", size[0]), ("v", size[1])):
        x = randn(pages, kv_heads, page, dim) * z
        if case["bits"] == 8:
            state[name + "_pages"], state[name + "_scale"] = eight_bit(x)
        else:
            state[name + "_pages"], state[name + "_scale"] = x.to(dtype), None
    if case["kind"] == "attention":
        return dict(state, q=randn(rows, heads * dim).to(dtype))
    proj = randn(rows, (heads + 2 * kv_heads) * dim).to(dtype)                            # one projection's columns
    freq = 10000.0 ** (-torch.arange(case["pairs"], dtype=torch.float64, device="cuda") / max(1, case["pairs"]))
    return dict(state, q=proj[:, :heads * dim], k=proj[:, heads * dim:(heads + kv_heads) * dim], v=proj[:, (heads + kv_heads) * dim:],
                freq=freq.float() if case["pairs"] else None)


# ---- one pass -----------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": own_append, "attention": own_attention, "adapter": own_adapter}[kind](state)
    return {"append": plain_append, "attention": plain_attention, "adapter": plain_adapter}[kind](state)


def own_append(s):
    from energonai_b200.paged import paged_append
    q = paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["tables"], s["starts"], s["lengths"], s["most_new"], freq=s["freq"],
                     k_scale=s["k_scale"], v_scale=s["v_scale"])
    return appended(s, q)


def own_attention(s):
    from energonai_b200.paged import paged_attention
    return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["starts"], s["lengths"], s["most_new"], s["most_length"],
                           window=s["case"]["window"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def own_adapter(s):
    from energonai_b200.adapter import adapter_product
    return adapter_product(s["x"], s["w"], s["a"], s["b"], s["scales"], s["index"], s["starts"], s["most_new"], bias=s["bias"])


def appended(s, q):
    return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def padded(s):
    """Row of token i of sequence b, [batch, most_new], and which of them there are."""
    i = torch.arange(s["most_new"], device="cuda")[None, :]
    starts = s["starts"].long()
    there = i < (starts[1:] - starts[:-1])[:, None]
    return torch.where(there, starts[:-1, None] + i, 0), there


def positions(s):
    """Position of token i of sequence b, [batch, most_new]."""
    starts = s["starts"].long()
    return (s["lengths"] - (starts[1:] - starts[:-1]))[:, None] + torch.arange(s["most_new"], device="cuda")[None, :]


def rotated(x, angle):
    """Rows x [rows, heads, dim] with their leading pairs turned by angle [rows, pairs]."""
    n = 2 * angle.shape[1]
    even, odd = x[..., 0:n:2], x[..., 1:n:2]
    c, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turned = torch.stack([even * c - odd * sn, odd * c + even * sn], -1).flatten(-2)
    return torch.cat([turned, x[..., n:]], -1)


def plain_append(s):
    c, dtype = s["case"], s["q"].dtype
    page, kv_heads, dim = c["page"], c["kv_heads"], c["dim"]
    at, there = padded(s)
    pos = positions(s)
    q, k, v = (s[n].float().unflatten(1, (-1, dim)) for n in "qkv")
    if s["freq"] is not None:
        angle = pos[there].double()[:, None] * s["freq"].double()[None, :]
        q, k = rotated(q, angle), rotated(k, angle)
    first = pos[:, :1] // page                                         # the first page that a sequence writes
    here = torch.where(there, pos // page - first, -1)
    count = (s["most_new"] - 1) // page + 2
    written = torch.zeros((c["batch"], count, page), dtype=torch.bool, device="cuda")
    b = torch.arange(c["batch"], device="cuda")[:, None].expand_as(pos)[there]
    spot = (b, here[there], pos[there] % page)
    written[spot] = True
    touched = written.any(-1)
    ids = s["tables"].long().gather(1, (first + torch.arange(count, device="cuda")[None, :]).clamp(max=s["tables"].shape[1] - 1))[touched]
    fresh = written[..., 0][touched]
    for x, pages, scale in ((k, s["k_pages"], s["k_scale"]), (v, s["v_pages"], s["v_scale"])):
        rows = torch.zeros((c["batch"], count, page, kv_heads, dim), device="cuda")
        rows[spot] = x[at[there]]
        rows = rows[touched].transpose(1, 2)                           # [pages, kv_heads, page, dim]
        fill = written[touched][:, None, :, None]
        if scale is None:
            pages[ids] = torch.where(fill, rows.to(dtype), pages[ids])
            continue
        m, e = torch.frexp(rows.abs().amax((-2, -1)))                  # the smallest 2^k with amax <= 448 * 2^k
        need = torch.exp2((e - 9 + (m > 0.875)).clamp(min=-100).float())
        before = scale[ids]
        after = torch.where(fresh[:, None], need, torch.maximum(before, need))
        old = pages[ids].float()
        kept = old * (before / after)[..., None, None]
        earlier = (torch.arange(page, device="cuda")[None, :] < written[touched].int().argmax(-1)[:, None])[:, None, :, None]
        value = torch.where(fill, rows / after[..., None, None], torch.where(earlier, kept, old))
        pages[ids] = value.to(E4M3)
        scale[ids] = after
    return appended(s, q.flatten(1).to(dtype))


def plain_attention(s):
    c, dtype = s["case"], s["q"].dtype
    batch, heads, kv_heads, dim = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    at, there = padded(s)
    q = s["q"].float()[at].view(batch, s["most_new"], kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)

    def gathered(pages, scale):
        x = pages[s["tables"].long()].float()                          # [batch, pages, kv_heads, page, dim]
        if scale is not None:
            x *= scale[s["tables"].long()][..., None, None]
        return x.transpose(1, 2).flatten(2, 3)

    score = q @ gathered(s["k_pages"], s["k_scale"]).transpose(2, 3) * dim ** -0.5
    key = torch.arange(score.shape[-1], device="cuda")
    pos = positions(s)[:, :, None]
    seen = key <= pos
    if c["window"]:
        seen &= key > pos - c["window"]
    score = score.unflatten(2, (heads // kv_heads, -1)).masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    weight = score.exp_()
    weight /= weight.sum(-1, keepdim=True)
    out = weight.flatten(2, 3) @ gathered(s["v_pages"], s["v_scale"])
    out = out.unflatten(2, (heads // kv_heads, -1)).permute(0, 3, 1, 2, 4).flatten(2)
    return out[there].to(dtype)


def plain_adapter(s):
    at, there = padded(s)
    x = s["x"].float()
    y = x @ s["w"].float().T
    if s["bias"] is not None:
        y += s["bias"].float()
    index = s["index"].long().clamp(min=0)
    scale = torch.where(s["index"] >= 0, s["scales"][index], 0.0)[:, None, None]
    low = x[at] @ s["a"][index].float().transpose(1, 2) * scale
    y += (low @ s["b"][index].float().transpose(1, 2))[there]
    return y.to(s["x"].dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    new, length = lengths(case)
    begin = [sum(new[:b]) for b in range(len(new))]
    if case["kind"] == "adapter":
        y = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        for b, i in enumerate(s["index"].tolist()):
            if i >= 0:
                r = slice(begin[b], begin[b] + new[b])
                y[r] += float(s["scales"][i]) * torch.einsum("mk,rk,nr->mn", s["x"][r].double(), s["a"][i].double(), s["b"][i].double())
        return y + s["bias"].double() if case["bias"] else y
    page, heads, kv_heads, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    table = s["tables"].tolist()
    if case["kind"] == "attention":
        out = torch.empty((sum(new), kv_heads, heads // kv_heads, dim), dtype=torch.float64, device="cuda")
        for b, n in enumerate(length):
            ids = torch.tensor(table[b][:-(-n // page)], device="cuda")
            lo = max(0, n - new[b] - case["window"] + 1) if case["window"] else 0
            for g in range(kv_heads):
                k, v = ((p[ids, g].double() * (1 if z is None else z[ids, g].double()[:, None, None])).reshape(-1, dim)[lo:n]
                        for p, z in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
                q = s["q"][begin[b]:begin[b] + new[b]].double().view(new[b], kv_heads, -1, dim)[:, g]
                z = torch.einsum("ihd,jd->ihj", q, k) / math.sqrt(dim)
                distance = torch.arange(n - new[b], n, device="cuda")[:, None] - torch.arange(lo, n, device="cuda")[None, :]
                z[((distance < 0) | ((distance >= case["window"]) if case["window"] else False))[:, None, :].expand_as(z)] = -math.inf
                out[begin[b]:begin[b] + new[b], g] = torch.einsum("ihj,jd->ihd", torch.softmax(z, -1), v)
        return out.flatten(1)
    at = torch.cat([torch.arange(n - m, n, dtype=torch.float64, device="cuda") for m, n in zip(new, length)])
    q, k, v = (s[x].double().view(sum(new), -1, dim).clone() for x in "qkv")
    if case["pairs"]:
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at[:, None] * s["freq"].double())
        for x in (q, k):
            pairs = torch.view_as_complex(x[..., :2 * case["pairs"]].unflatten(-1, (-1, 2)).contiguous()) * turn[:, None]
            x[..., :2 * case["pairs"]] = torch.view_as_real(pairs).flatten(-2)
    result = dict(q=q.flatten(1))
    for name, x in (("k", k), ("v", v)):
        pages = s[name + "_pages"].double()
        scale = None if case["bits"] == 16 else s[name + "_scale"].double()
        for b, n in enumerate(length):
            p = n - new[b]
            while p < n:
                i, slot = table[b][p // page], p % page
                more = min(page - slot, n - p)
                y = x[begin[b] + p - (n - new[b]):][:more].transpose(0, 1)
                if scale is not None:
                    need = torch.exp2(torch.ceil(torch.log2(y.abs().amax((1, 2)) / 448)))
                    if slot:
                        need = torch.maximum(need, scale[i])
                        pages[i, :, :slot] *= (scale[i] / need)[:, None, None]
                    scale[i] = need
                    y = y / need[:, None, None]
                pages[i, :, slot:slot + more] = y
                p += more
        result[name + "_pages"], result[name + "_scale"] = pages, scale
    return result


# ---- what a pass cannot do without --------------------------------------------------------------------------
def work(case):
    new, length = lengths(case)
    rows = sum(new)
    if case["kind"] == "adapter":
        width, columns, rank = case["width"], case["columns"], case["rank"]
        used = min(case["adapters"], case["batch"])
        return dict(bytes=2 * (rows * (width + columns) + width * columns + used * rank * (width + columns)),
                    flops=2 * rows * (width * columns + rank * (width + columns)))
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    held = case["bits"] // 8
    if case["kind"] == "append":
        return dict(bytes=rows * dim * ((4 * heads if case["pairs"] else 0) + 2 * kv_heads * (2 + held)), flops=rows * 3 * 2 * case["pairs"] * (heads + kv_heads))
    keys = pairs = 0
    for n, m in zip(new, length):
        lo = max(0, m - n - case["window"] + 1) if case["window"] else 0
        keys += m - lo
        pairs += sum(min(p + 1, case["window"] or p + 1) for p in range(m - n, m))
    return dict(bytes=4 * rows * heads * dim + 2 * keys * kv_heads * dim * held, flops=4 * pairs * heads * dim)
