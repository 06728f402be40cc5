"""Paged caches restated in 64 bits on the CPU: what new tokens leave in the pages, and what they attend to."""
import math
import random

import torch

E4M3 = torch.float8_e4m3fn
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, E4M3: 2.0 ** -4}       # half a step, relative


class Case:
    """A packed batch over pools of random pages.  Everything that no token may see is NaN: other pages, slots behind a
    sequence's last position; the tables end in numbers that are no pages."""

    def __init__(self, new, past, heads, kv_heads, dim, page, dtype, bits, seed=0, spare=2, pad_rows=0, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        r = random.Random(seed)
        self.new, self.length = list(new), [n + p for n, p in zip(new, past)]
        self.past, self.heads, self.kv_heads, self.dim, self.page, self.dtype, self.bits = list(past), heads, kv_heads, dim, page, dtype, bits
        need = [-(-n // page) for n in self.length]
        self.pages = sum(need) + spare
        order = r.sample(range(self.pages), self.pages)
        self.tables = []
        for n in need:
            self.tables.append(order[:n])
            order = order[n:]
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + pad_rows
        rnd = lambda *shape: torch.randn(*shape, generator=g)
        self.q = (rnd(self.rows, heads * dim) * magnitude).to(dtype)
        self.k, self.v = ((rnd(self.rows, kv_heads * dim) * magnitude).to(dtype) for _ in range(2))
        self.pool, self.scale = [], []
        for _ in range(2):
            x = rnd(self.pages, kv_heads, page, dim) * torch.exp2(torch.randint(-3, 4, (self.pages, kv_heads, 1, 1), generator=g).float())
            there = torch.zeros(self.pages, page, dtype=torch.bool)
            for t, n in zip(self.tables, self.length):
                for i, p in enumerate(t):
                    there[p, :n - i * page] = True
            if bits == 8:
                s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((-2, -1)) / 448)))
                codes = (x / s[..., None, None]).to(E4M3)
                codes.view(torch.uint8)[~there[:, None, :].expand(-1, kv_heads, -1)] = 0x7f
                self.pool.append(codes)
                self.scale.append(s)
            else:
                x = x.to(dtype)
                x[~there[:, None, :].expand(-1, kv_heads, -1)] = float("nan")
                self.pool.append(x)
                self.scale.append(None)

    def device(self, bad=-1):
        """(q, k, v), pools, scales, and the batch as tensors on the GPU."""
        cols = max(1, max(len(t) for t in self.tables)) + 1
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        tables = i32([t + [bad] * (cols - len(t)) for t in self.tables])
        up = lambda t: None if t is None else t.cuda()
        return [t.cuda() for t in (self.q, self.k, self.v)], [t.cuda() for t in self.pool], [up(t) for t in self.scale], (tables, i32(self.starts), i32(self.length), max(1, max(self.new)))

    def values(self, which, b):
        """Keys (0) or values (1) of sequence b, [length, kv_heads, dim] in 64 bits."""
        ids = torch.tensor(self.tables[b], dtype=torch.long)
        x = self.pool[which][ids].double()
        if self.bits == 8:
            x = x * self.scale[which][ids].double()[..., None, None]
        return x.transpose(1, 2).flatten(0, 1)[:self.length[b]]

    def attention(self, scale=None, window=0, prompt=1 << 30, missing=()):
        """(out, tolerance), [rows, heads*dim]; rows behind the last sequence are zero.

        The tolerance per element: the result's own rounding, u |o|; weights rounded to the products' type (fp16 2^-11; two bf16
        pieces 2^-16) once in the sum over values and, in effect, once in the sum of weights, 2 u_p sum w |v|; a score is a sum
        of `dim` products in fp32, at most 16 of which (one per 16 dimensions, truncated) are rounded into the accumulator, 2^-19
        sum |q||k| scale, and its exponential is off by 2^-18 at most, both once above and once below.  fp16 weights are
        held as 2^6 and more times their share of the row's largest weight; where they fall below fp16's normal range all the same, they are off by
        2^-25, that is 2^-31 of a share at most: 2^-31 sum |v|.  A result below fp16's normal range is off by 2^-25.  Sequences with more than `prompt`
        new tokens take the prompt kernel, whose bf16 weights over 16-bit pages are rounded once, 2^-8.  missing: table entries of pages
        that are none."""
        scale = self.dim ** -0.5 if scale is None else scale
        out, tol = torch.zeros(self.rows, self.heads, self.dim, dtype=torch.float64), torch.zeros(self.rows, self.heads, self.dim, dtype=torch.float64)
        group = self.heads // self.kv_heads
        for b, n in enumerate(self.new):
            if not n:
                continue
            u_p = 2.0 ** -11 if self.bits == 8 or self.dtype == torch.float16 else 2.0 ** -8 if n > prompt else 2.0 ** -16
            rows = slice(self.starts[b], self.starts[b] + n)
            k, v = (self.values(i, b).repeat_interleave(group, 1) for i in (0, 1))
            q = self.q[rows].double().view(n, self.heads, self.dim)
            s = torch.einsum("ihd,jhd->hij", q, k) * scale
            size = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * scale
            pos, key = torch.arange(self.past[b], self.length[b])[:, None], torch.arange(self.length[b])[None]
            seen = (key <= pos) & ((key > pos - window) if window else torch.ones(()).bool())
            for at in missing:
                seen = seen & ((key < at * self.page) | (key >= (at + 1) * self.page))
            w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            delta = 2.0 ** -19 * size.masked_fill(~seen, 0).amax(-1) + 2.0 ** -18
            o = torch.einsum("hij,jhd->ihd", w, v)
            size = torch.einsum("hij,jhd->ihd", w, v.abs())
            out[rows] = o
            tol[rows] = UNIT[self.dtype] * o.abs() + (2 * u_p + 2 * delta.T[..., None]) * size
            if self.bits == 8 or self.dtype == torch.float16:
                tol[rows] += 2.0 ** -31 * torch.einsum("hij,jhd->ihd", seen.expand(w.shape).double(), v.abs())
            if self.dtype == torch.float16:
                tol[rows] += 2.0 ** -25
        return out.flatten(1), tol.flatten(1)

    def turned(self, x, freq):
        """Rows [rows, n*dim] turned by their positions; and what 32-bit arithmetic may be off by: the angle's remainder, sine and cosine
        are each off by 2^-23 at most, a product and a sum by 2^-24 each: 2^-21 of the pair's length bounds all of them."""
        x = x.double().view(self.rows, -1, self.dim).clone()
        slack = torch.zeros_like(x)
        if freq is not None:
            at = torch.cat([torch.arange(p, n, dtype=torch.float64) for p, n in zip(self.past, self.length)] + [torch.zeros(self.rows - self.starts[-1], dtype=torch.float64)])
            angle = (at[:, None] * freq.double())[:, None]
            n = 2 * freq.numel()
            a, b = x[..., 0:n:2].clone(), x[..., 1:n:2].clone()
            x[..., 0:n:2], x[..., 1:n:2] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
            slack[..., :n] = (2.0 ** -21 * torch.hypot(a, b)).repeat_interleave(2, -1)
        return x, slack

    def append(self, freq=None):
        """The pools (value, tolerance, scale) after the new tokens, in 64 bits; and the queries (value, tolerance)."""
        q, slack = self.turned(self.q, freq)
        result = [(q.flatten(1), (UNIT[self.dtype] * (q.abs() + slack) + slack).flatten(1) if freq is not None else torch.zeros_like(q).flatten(1))]
        for which, x in ((0, self.k), (1, self.v)):
            x, slack = self.turned(x, freq if which == 0 else None)
            pool = self.pool[which].double()
            if self.bits == 8:
                pool = pool * self.scale[which].double()[..., None, None]
            tol = torch.zeros_like(pool)
            scale = self.scale[which].clone() if self.bits == 8 else None
            for b, n in enumerate(self.new):
                for at in range(self.past[b] // self.page, -(-self.length[b] // self.page) if n else 0):
                    page, begin, end = self.tables[b][at], max(at * self.page, self.past[b]), min((at + 1) * self.page, self.length[b])
                    rows = slice(self.starts[b] + begin - self.past[b], self.starts[b] + end - self.past[b])
                    slot = begin - at * self.page
                    y, s = x[rows].transpose(0, 1), slack[rows].transpose(0, 1)
                    new = slice(slot, slot + end - begin)
                    pool[page, :, new], tol[page, :, new] = y, s
                    if scale is None:
                        tol[page, :, new] += (UNIT[self.dtype] * (y.abs() + s)) * (freq is not None and which == 0)
                        continue
                    finite = torch.where(torch.isfinite(y), y.abs(), 0.0).amax((1, 2))
                    need = torch.exp2(torch.ceil(torch.log2(finite / 448)).clamp(min=-100)).float()
                    if slot:
                        need = torch.maximum(need, scale[page])
                        grown = (need > scale[page])[:, None, None]
                        old = pool[page, :, :slot]
                        tol[page, :, :slot] = torch.where(grown, torch.maximum(2.0 ** -4 * old.abs(), 2.0 ** -10 * need.double()[:, None, None]), 0.0)
                    scale[page] = need
                    # half a step: relative, or of the subnormal numbers, 2^-10 of the scale
                    tol[page, :, new] += torch.maximum(UNIT[E4M3] * (y.abs() + s), 2.0 ** -10 * need.double()[:, None, None])
            result.append((pool, tol, scale))
        return result
