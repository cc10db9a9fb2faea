"""Plain 64-bit forms of windowed attention, rotation and compaction for the GPU tests,
and how far a 32-bit computation rounded once may be from them."""
import math

import numpy as np
import torch

from chibillm_amd import ckv

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half a step of each type, relative to the value
ROUND = {t: torch.finfo(t).eps / 2 for t in DTYPES.values()}
STEP32 = 2.0 ** -23


def seen(position, window, sinks):
    """Tokens a row at `position` attends, in order."""
    t = np.arange(position + 1)
    return t[(t > position - window) | (t < sinks)]


def attention(q, k, v, rows, scale, p_bits=32):
    """q [rows, q_heads, d], k and v [tokens, kv_heads, d], rows: the tokens each row
    attends. Returns the output in 64 bits and the bound of its error before the one
    rounding to the output's type.

    A score's products are summed in 32 bits: off by at most (d + 8) steps of the sum
    of their magnitudes, for any order. An error of e in every score moves a
    probability by at most 2e of itself (e in its exponent and e in the sum), as does
    each step of the exponential, the sum and the division; with n keys the weighted sum
    of values adds n steps of their largest. p_bits: significant bits that enter the
    product with v."""
    rows_n, heads, d = q.shape
    h = k.shape[1]
    out = torch.zeros(rows_n, heads, d, dtype=torch.float64)
    bound = torch.zeros(rows_n, heads, 1, dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for r, t in enumerate(rows):
        for head in range(heads):
            kk, vv = k[t, head // (heads // h)], v[t, head // (heads // h)]
            s = kk @ q[r, head] * scale
            p = torch.softmax(s, 0)
            out[r, head] = p @ vv
            e = (d + 8) * STEP32 * float((kk.abs() @ q[r, head].abs()).max()) * abs(scale)
            big = float(s.abs().max()) + 1  # the exponent's own rounding grows with the score
            relative = 2 * e + (8 + 2 * big + 2 * len(t)) * STEP32 + 2.0 ** (1 - p_bits)
            bound[r, head] = relative * float(vv.abs().max())
    return out, bound


def assert_within(got, want, bound, what):
    """`got` in its type against `want` in 64 bits: the bound and one rounding."""
    got64, want = got.detach().cpu().double(), want.cpu()
    room = bound * (1 + ROUND[got.dtype]) + ROUND[got.dtype] * want.abs()
    if got.dtype == torch.float16:
        room = room + 2.0 ** -25  # half of its smallest step
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got64), finite), f"{what}: other values are finite"
    off = ((got64 - want).abs() - room)[finite]
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, f"{what}: off by {worst:.3g} more than the bound"


def turned(x, angle, rotary):
    """x [rows, heads, d] in 64 bits, pair j of every head by angle[row, j]."""
    x = x.double().clone()
    a, b = x[..., :rotary // 2].clone(), x[..., rotary // 2:rotary].clone()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    x[..., :rotary // 2], x[..., rotary // 2:rotary] = a * c - b * s, b * c + a * s
    return x


def turned_bound(x, rotary):
    """Error of `turned` in 32 bits before its rounding: sine and cosine are within two
    steps of theirs (and 1e-9), each product and the sum within half a step."""
    x = x.double().abs()
    pair = (x[..., :rotary // 2] + x[..., rotary // 2:rotary]) * (4 * STEP32)
    return torch.cat([pair, pair, torch.zeros_like(x[..., rotary:])], -1)


def frequencies(theta, rotary):
    return torch.tensor([float(np.float32(theta)) ** (-2.0 * j / rotary) for j in range(rotary // 2)],
                        dtype=torch.float64)


class Cache:
    """A pool of one test: scattered pages that hold NaN wherever nothing was written, and a
    host copy of what was. Tables are kept per sequence."""

    def __init__(self, ctx, dtype, lengths, kv_heads, head_dim, page=16, layers=1, spare=3, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.dtype, self.page, self.h, self.d = DTYPES[dtype], page, kv_heads, head_dim
        pages = [-(-n // page) for n in lengths]
        self.blocks = sum(pages) + spare
        order = torch.randperm(self.blocks, generator=self.g).numpy().astype(np.uint32)
        self.tables = np.split(order[:sum(pages)], np.cumsum(pages)[:-1])
        self.free = order[sum(pages):]  # pages no sequence holds
        self.lengths = list(lengths)
        shape = (layers, self.blocks * page, kv_heads, head_dim)
        self.k = torch.full(shape, math.nan, dtype=self.dtype)
        self.v = self.k.clone()
        for t, n in zip(self.tables, lengths):
            at = torch.from_numpy(self.slots(t, np.arange(n)))
            self.k[:, at], self.v[:, at] = self.randn(layers, n, kv_heads, head_dim), self.randn(layers, n, kv_heads, head_dim)
        self.ctx, self.layers = ctx, layers

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype)

    def slots(self, table, tokens):
        tokens = np.asarray(tokens)
        return np.asarray(table)[tokens // self.page].astype(np.int64) * self.page + tokens % self.page

    def to_device(self):
        self.kd, self.vd = self.k.cuda(), self.v.cuda()
        self.pool = ckv.Pool(self.ctx, self.layers, self.blocks, self.page, self.h, self.d, self.dtype,
                             self.kd.view(-1), self.vd.view(-1))
        return self.pool

    def upload(self, first, counts, slots=True):
        """Rows first[s] .. first[s] + counts[s] - 1 of every sequence."""
        flat = np.concatenate(self.tables)
        starts = np.cumsum([0] + [t.size for t in self.tables[:-1]])
        seq = np.repeat(np.arange(len(self.tables)), counts)
        pos = np.concatenate([np.arange(f, f + c) for f, c in zip(first, counts)])
        at = np.array([self.slots(self.tables[s], [p])[0] for s, p in zip(seq, pos)])
        self.pool.upload(flat, starts[seq], [self.tables[s].size for s in seq], pos, at if slots else None)
        return seq, pos, at

    def unchanged(self, but=()):
        """Nothing but the slots `but` changed, bit for bit (NaN included)."""
        ints = {2: torch.int16, 4: torch.int32}[self.k.element_size()]
        keep = np.setdiff1d(np.arange(self.blocks * self.page), np.asarray(but))
        for dev, host in ((self.kd, self.k), (self.vd, self.v)):
            assert torch.equal(dev.cpu().view(ints)[:, keep], host.view(ints)[:, keep])
