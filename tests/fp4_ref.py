"""Plain 64-bit forms of 4-bit caches, scaled rotations and attention for the GPU tests, how far
the computed ones may be from them, and a cache of a test's own."""
import math

import numpy as np
import torch

from chibillm_amd import ckv
from tests.operator_ref import DTYPES, ROUND, STEP32

LEAST = {"f16": -23, "bf16": -100, "f32": -100}
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
# magnitudes from which on a code is taken: halfway to the next level, the tie to the even code
BORDERS = [(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)]


def held(x, dtype):
    """x [..., 32 n] in 64 bits as a 4-bit pool of rows of `dtype` holds it."""
    y = x.double().unflatten(-1, (-1, 32))
    largest = y.abs().amax(-1, keepdim=True)
    lost = ~(largest < 2.0 ** (16 if dtype == "f16" else 128))
    exponent = torch.frexp(torch.where(lost, 1.0, largest)).exponent - 3
    exponent = torch.where(largest == 0, LEAST[dtype], exponent).clamp(min=LEAST[dtype])
    scale = torch.ldexp(torch.ones_like(largest), exponent)
    a = (y / scale).abs()
    code = sum(((a >= b) if tie else (a > b)).long() for b, tie in BORDERS)
    out = torch.copysign(LEVELS[code], y) * scale
    return torch.where(lost, math.nan, out).flatten(-2)


def frequencies(rotation, d):
    """Turns of each pair per position, in 80 bits."""
    r = rotation.rotary_dim or d
    j = np.arange(r // 2, dtype=np.longdouble)
    whole = 2 * np.longdouble("3.14159265358979323846264338327950288")
    theta, factor = np.longdouble(rotation.theta), np.longdouble(rotation.factor)
    b = theta ** (-2 * j / r)
    if rotation.scaling == 1:
        b = b / factor
    low, high, original = np.longdouble(rotation.low), np.longdouble(rotation.high), np.longdouble(rotation.original)
    if rotation.scaling == 2:
        keep = np.clip((original * b / whole - low) / (high - low), 0, 1)
        b = b * (keep + (1 - keep) / factor)
    if rotation.scaling == 3:
        at = lambda turns: r * np.log(original / (turns * whole)) / (2 * np.log(theta))
        first, last = max(np.floor(at(high)), 0), min(np.ceil(at(low)), r - 1)
        mix = np.clip((j - first) / max(last - first, np.longdouble("0.001")), 0, 1)
        b = b * (1 - mix) + b / factor * mix
    return b / whole


def magnitude(rotation):
    if rotation.magnitude:
        return float(rotation.magnitude)
    factor = float(rotation.factor)
    return 0.1 * math.log(factor) + 1 if rotation.scaling == 3 and factor > 1 else 1.0


def rotated(x, positions, rotation, angle_error=0.0):
    """x [rows, heads, d] in 64 bits at `positions`, and the error of a 32-bit rotation before its
    rounding: sine and cosine within two steps, products and their sum half a step each, the
    magnitude another; and of angles off by `angle_error` of themselves."""
    d = x.shape[-1]
    r = rotation.rotary_dim or d
    turn = np.asarray(positions, np.longdouble)[:, None] * frequencies(rotation, d)
    angle = torch.from_numpy(((turn - np.floor(turn)) * 2 * np.longdouble("3.14159265358979323846264338327950288")).astype(np.float64))
    m = magnitude(rotation)
    c, s = (angle.cos() * m)[:, None], (angle.sin() * m)[:, None]
    y = x.double().cpu().clone()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if rotation.layout == 0 else (slice(0, r, 2), slice(1, r, 2))
    a, b = y[..., first].clone(), y[..., second].clone()
    room = torch.zeros_like(y)
    off = torch.from_numpy((turn * 2 * np.pi).astype(np.float64))[:, None] * angle_error
    room[..., first] = room[..., second] = (a.abs() + b.abs()) * m * (6 * STEP32 + off)
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y, room


def attention(q, k, v, seen, scale, q_half=0.0, p_half=0.0, p_floor=0.0):
    """q [rows, q_heads, d], k and v [tokens, kv_heads, d], seen: how many of the tokens each row
    attends. Returns the output in 64 bits and the bound of its error before the one rounding.

    Scores: products summed in 32 bits, off by at most (d + 8) steps of the sum of their
    magnitudes in any order, and queries kept to `q_half` of themselves. An error of e in every
    score moves a probability by at most 2e of itself; the exponential, the sums and the division
    add steps; p_half: half a step of the type that probabilities enter the product with v in,
    p_floor: half its smallest number (of the row's largest probability)."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for head in range(heads):
        kk, vv, qq = k[:, head // group], v[:, head // group], q[:, head]
        for r in range(n):
            t = int(seen[r])
            s = kk[:t] @ qq[r] * scale
            p = torch.softmax(s, 0)
            out[r, head] = p @ vv[:t]
            e = ((d + 8) * STEP32 + q_half) * float((kk[:t].abs() @ qq[r].abs()).max()) * abs(scale)
            relative = 2 * e + (8 + 2 * (float(s.abs().max()) + 1) + 2 * t) * STEP32 + 2 * p_half
            bound[r, head] = relative * (p @ vv[:t].abs()) + t * p_floor * float(p.max()) * vv[:t].abs().amax(0)
    return out, bound


# what attention keeps of its operands: 16 bits of queries and probabilities in decode rows
# (bf16 terms), the rows' type in tiles, and 24 bits where rows are floats
def decode_bits(dtype):
    return {"q_half": STEP32, "p_half": STEP32} if dtype == "f32" else {"q_half": 2.0 ** -17, "p_half": 2.0 ** -17}


def tile_bits(dtype):
    if dtype == "f32":
        return {"p_half": STEP32}
    return {"p_half": ROUND[DTYPES[dtype]], "p_floor": 2.0 ** -25 if dtype == "f16" else 0.0}


def assert_within(got, want, bound, what):
    """`got` in its type against `want` in 64 bits: the bound and one rounding."""
    g = got.detach().cpu().double().reshape(want.shape)
    room = bound * (1 + ROUND[got.dtype]) + ROUND[got.dtype] * want.abs()
    if got.dtype == torch.float16:
        room = room + 2.0 ** -25  # half of its smallest number
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(g), finite), f"{what}: other values are finite"
    off = ((g - want).abs() - room)[finite]
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, f"{what}: off by {worst:.3g} more than the bound"


def gated(out, bound, gate):
    """Times the sigmoid of a gate, which 32 bits compute to 8 steps."""
    g = torch.sigmoid(gate.double().cpu())
    return out * g, (bound + 8 * STEP32 * out.abs()) * g


class Cache:
    """A 4-bit pool of one test over scattered pages, wherever nothing was written full of bytes that
    read as NaN, and a host copy in 64 bits of what it should hold."""

    def __init__(self, ctx, dtype, lengths, kv_heads, head_dim, page=16, layers=1, spare=3, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.name, self.dtype, self.page, self.h, self.d = dtype, DTYPES[dtype], page, kv_heads, head_dim
        pages = [-(-n // page) for n in lengths]
        self.blocks = sum(pages) + spare
        order = torch.randperm(self.blocks, generator=self.g).numpy().astype(np.uint32)
        self.tables = np.split(order[:sum(pages)], np.cumsum(pages)[:-1])
        self.starts = np.concatenate([[0], np.cumsum(pages)[:-1]]).astype(int)
        self.lengths, self.free = list(lengths), order[sum(pages):]
        size = layers * self.blocks * page * kv_heads * head_dim * 17 // 32
        self.bytes = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.pool = ckv.Pool(ctx, layers, self.blocks, page, kv_heads, head_dim, self.dtype, *self.bytes, fp4=True)
        shape = (layers, self.blocks * page, kv_heads, head_dim)
        self.k = torch.full(shape, math.nan, dtype=torch.float64)
        self.v = self.k.clone()

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype)

    def slots(self, i, positions):
        p = np.asarray(positions, int)
        return self.tables[i][p // self.page].astype(np.int64) * self.page + p % self.page

    def upload(self, first, counts, with_slots=True):
        """A batch of `counts` rows of each sequence from position `first`; their slots."""
        rows = [(i, p) for i, (f, c) in enumerate(zip(first, counts)) for p in range(f, f + c)]
        seq = np.array([i for i, _ in rows], int)
        positions = np.array([p for _, p in rows], int)
        at = np.concatenate([self.slots(i, range(f, f + c)) for i, (f, c) in enumerate(zip(first, counts))])
        lengths = np.array([t.size for t in self.tables])
        self.pool.upload(np.concatenate(self.tables), self.starts[seq], lengths[seq], positions, at if with_slots else None)
        self.rows, self.at = rows, torch.from_numpy(at)
        return positions

    def keep(self, layer, k, v, at=None):
        """The rows (64 bits, or the type's) as the pool should hold them."""
        at = self.at if at is None else at
        for cache, x in ((self.k, k), (self.v, v)):
            cache[layer, at] = held(x.double().cpu().reshape(len(at), -1), self.name).reshape(len(at), self.h, self.d)

    def fill(self, layer=0, make=None):
        """Every token of every sequence appended in one batch."""
        self.upload([0] * len(self.lengths), self.lengths)
        k, v = (make or self.randn)(len(self.rows), self.h, self.d), (make or self.randn)(len(self.rows), self.h, self.d)
        self.pool.append(layer, k.cuda().flatten(1), v.cuda().flatten(1))
        self.keep(layer, k, v)
        return k, v

    def read(self, layer=0):
        """Keys and values of all tokens of all sequences, as the pool reads them."""
        got = []
        for i, n in enumerate(self.lengths):
            out = [torch.zeros(n, self.h * self.d, dtype=self.dtype, device="cuda") for _ in range(2)]
            self.pool.gather(layer, int(self.starts[i]), self.tables[i].size, n, *out)
            got.append(out)
        return [torch.cat([x[s] for x in got]).cpu().reshape(-1, self.h, self.d) for s in range(2)]

    def should(self, layer=0):
        at = torch.from_numpy(np.concatenate([self.slots(i, range(n)) for i, n in enumerate(self.lengths)]))
        return self.k[layer, at], self.v[layer, at]

    def check(self, layer=0, what=""):
        for got, want, name in zip(self.read(layer), self.should(layer), ("keys", "values")):
            got = got.double()
            assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what} {name}: other numbers are NaN"
            assert torch.equal(got.nan_to_num(), want.nan_to_num()), f"{what} {name}"
            assert torch.equal(torch.signbit(got)[~torch.isnan(want)], torch.signbit(want)[~torch.isnan(want)])

    def attended(self, q, scale, layer=0, **bits):
        """The batch's rows [rows, q_heads, d] attended in 64 bits, and the bound."""
        q, out, bound = q.double().cpu(), [], []
        for i in range(len(self.lengths)):
            mine = [r for r, (s, _) in enumerate(self.rows) if s == i]
            if not mine:
                continue
            seen = [self.rows[r][1] + 1 for r in mine]
            at = torch.from_numpy(self.slots(i, range(max(seen))))
            o, b = attention(q[mine], self.k[layer, at], self.v[layer, at], seen, scale, **bits)
            out.append(o)
            bound.append(b)
        return torch.cat(out), torch.cat(bound)
