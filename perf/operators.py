"""Operators of a serving program whose context outgrows its cache, as calls to measure.

A layer that attends through a window keeps a few first tokens (sinks) in sight and
reads only the window's pages besides; a cache that is full drops tokens and moves the
kept ones together, turning their keys to their new positions; tokens of images and
video carry a position on several axes. The cases are single calls of these on a paged
pool whose pages are scattered, as a serving program has it. Values are N(0, 1) from
the seed.

`own` false computes a call in elementary torch operations, true calls `chibillm_amd.ckv`;
`exact` answers in 64 bits.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# Heads of one attention layer. "narrow": the KV shape of the benchmark's model (8 kv
# heads of 128, 16 query heads, rotary over the whole head). "wide": a layer with an
# output gate, 256-wide heads in groups of four and rotary on a quarter of the head.
NARROW = {"kv_heads": 8, "q_heads": 16, "head_dim": 128, "rotary": 128, "theta": 1e6, "gated": False}
WIDE = {"kv_heads": 2, "q_heads": 8, "head_dim": 256, "rotary": 64, "theta": 1e7, "gated": True}


def _case(op, heads, **more):
    return {"op": op, **heads, "dtype": "bf16", **more}


def listed():
    return [
        # the smallest call: four chats, most still shorter than the window, one layer of
        # one decode step, where launches and round trips count
        dict(_case("decode", NARROW, rows=4, low=60, high=1900, window=512, sinks=4), name="window decode 4 rows"),
        # an ordinary serving batch far past its window
        dict(_case("decode", NARROW, rows=48, low=900, high=12000, window=1024, sinks=4), name="window decode 48 rows"),
        # a gated layer with wide heads and a long window
        dict(_case("decode", WIDE, rows=24, low=200, high=9000, window=2048, sinks=16), name="window decode wide heads"),
        # the middle of a long prompt: one sequence's next chunk
        dict(_case("prefill", NARROW, sequences=1, rows_low=512, rows_high=512, prefix=6000, window=1024, sinks=4), name="window prefill one chunk"),
        # new prompts of mixed lengths batched together, a short window, no sinks
        dict(_case("prefill", NARROW, sequences=9, rows_low=17, rows_high=900, prefix=0, window=256, sinks=0, dtype="f16"), name="window prefill new prompts"),
        # the largest: many sequences' chunks at once, a long window
        dict(_case("prefill", NARROW, sequences=16, rows_low=1024, rows_high=1024, prefix=4000, window=2048, sinks=4), name="window prefill batch"),
        # pools in the storage type of the reference engine
        dict(_case("prefill", NARROW, sequences=2, rows_low=220, rows_high=300, prefix=1000, window=512, sinks=4, dtype="f32"), name="window prefill f32"),
        # a decode step of a few chats about images: time, height and width positions
        dict(_case("rotate", NARROW, rows=6, axes=3, mixed=True), name="axes decode rows"),
        # a prompt with large images: queries and keys rotated, keys and values appended
        dict(_case("rotate", NARROW, rows=4096, axes=3, mixed=False), name="axes image prompt"),
        # the wide layer's quarter-head rotary over a short video
        dict(_case("rotate", WIDE, rows=1531, axes=3, mixed=True, dtype="f16"), name="axes wide heads"),
        # a chat that reached its limit drops the older half of its middle: every layer's
        # kept tail moves down in place and its keys turn back
        dict(_case("compact", NARROW, sequences=1, low=2011, high=2011, layers=28, pattern="middle", fresh=False), name="compact one chat"),
        # a batch evicted token by token, its kept tokens gathered into other pages
        dict(_case("compact", NARROW, sequences=6, low=700, high=3500, layers=12, pattern="scattered", fresh=True), name="compact scattered batch"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges; none costs more than the largest listed one."""
    op = rng.choice(["decode"] * 3 + ["prefill"] * 3 + ["rotate"] * 2 + ["compact"] * 2)
    wide = rng.random() < 0.3
    heads = dict(WIDE if wide else NARROW)
    if wide:  # the same layer at other head counts of its kind
        heads["kv_heads"] = rng.choice([1, 2, 4])
        heads["q_heads"] = heads["kv_heads"] * rng.choice([2, 4])
        heads["gated"] = rng.random() < 0.7
    dtype = rng.choice(["bf16", "bf16", "f16"] + ([] if wide and op == "prefill" else ["f32"]))
    if op == "rotate":
        return _case(op, heads, rows=_log(rng, 1, 4096), axes=rng.choice([1, 2, 3, 3]), mixed=rng.random() < 0.5, dtype=dtype)
    if op == "compact":
        sequences, layers = rng.randint(1, 6), rng.choice([4, 12, 28])
        high = _log(rng, 40, min(3500, 90_000 // (layers * sequences)))
        return _case(op, heads, sequences=sequences, low=max(8, int(high * rng.uniform(0.2, 1.0))), high=high, layers=layers,
                     pattern=rng.choice(["middle", "scattered"]), fresh=rng.random() < 0.5, dtype=dtype)
    window, sinks = _log(rng, 17, 2048), rng.choice([0, 1, 4, 4, 16, 33])
    if op == "decode":
        rows = _log(rng, 1, 64)
        high = _log(rng, 40, max(64, min(16000, 400_000 // rows)))
        return _case(op, heads, rows=rows, low=max(1, int(high * rng.uniform(0.05, 1.0))), high=high, window=window, sinks=sinks, dtype=dtype)
    sequences = _log(rng, 1, 12 if dtype != "f32" else 3)
    high = _log(rng, 9, 1024 if dtype != "f32" else 400)
    return _case(op, heads, sequences=sequences, rows_low=max(2, int(high * rng.uniform(0.1, 1.0))), rows_high=high,
                 prefix=rng.choice([0, _log(rng, 3, 4000)]), window=window, sinks=sinks, dtype=dtype)


# ---- shapes of a case (the same for every seed) ----

def _spread(n, low, high):
    """n lengths spread evenly over [low, high], in a mixed order."""
    order = np.random.RandomState(n).permutation(n)
    return [int(x) for x in np.round(np.linspace(low, high, n))[order]] if n > 1 else [high]


def _kept(case, tokens):
    """Indices of the tokens of one sequence that a compaction keeps."""
    if case["pattern"] == "middle":  # the first four, and the newer half
        return np.concatenate([np.arange(4), np.arange(max(4, tokens // 2), tokens)])
    pick = np.random.RandomState(tokens).rand(tokens) < 0.6  # by a score of their own, the first four always
    pick[:4] = True
    return np.flatnonzero(pick)


class _Batch:
    """Tables, positions and slots of a case's rows, over pages in an order drawn from the seed."""

    def __init__(self, case, seed):
        op = case["op"]
        if op == "prefill":
            counts = _spread(case["sequences"], case["rows_low"], case["rows_high"])
            first = [case["prefix"]] * len(counts)
        elif op == "rotate":
            counts, first = [case["rows"]], [0]
        else:
            spans = _spread(case["sequences"] if op == "compact" else case["rows"], case["low"], case["high"])
            counts, first = [1] * len(spans), [n - 1 for n in spans]
        self.counts, self.first = counts, first
        spans = [f + c for f, c in zip(first, counts)]
        pages = [-(-n // PAGE) for n in spans]
        if op == "compact":  # the pages the kept tokens go to, where they are others
            self.kept = [_kept(case, n) for n in spans]
            pages += [-(-x.size // PAGE) for x in self.kept] if case["fresh"] else []
        self.blocks = sum(pages) + 5
        order = np.random.RandomState(seed % (1 << 32)).permutation(self.blocks).astype(np.uint32)
        self.tables = np.split(order[:sum(pages)], np.cumsum(pages)[:-1])
        if op == "compact":
            targets = self.tables[len(spans):] if case["fresh"] else self.tables
            self.source = np.concatenate([self._slot(t, x) for t, x in zip(self.tables, self.kept)])
            self.target = np.concatenate([self._slot(t, np.arange(x.size)) for t, x in zip(targets, self.kept)])
            self.shift = np.concatenate([np.arange(x.size) - x for x in self.kept]).astype(np.int32)
            return
        seq = np.repeat(np.arange(len(spans)), counts)
        self.positions = np.concatenate([np.arange(f, f + c) for f, c in zip(first, counts)]).astype(np.uint32)
        self.flat = np.concatenate(self.tables)
        starts = np.concatenate([[0], np.cumsum(pages)[:-1]])
        self.starts = starts
        self.offsets = starts[seq].astype(np.uint32)
        self.lengths = np.array(pages, np.uint32)[seq]
        page = self.flat[self.offsets + self.positions // PAGE]
        self.slots = (page.astype(np.uint64) * PAGE + self.positions % PAGE).astype(np.uint32)
        if op == "rotate":
            self.axes, self.pair_axis = _axes(case)

    @staticmethod
    def _slot(table, index):
        return (table[index // PAGE].astype(np.int64) * PAGE + index % PAGE).astype(np.uint32)


def _axes(case):
    """Positions of the rows on each axis, and the axis that each rotary pair turns by."""
    rows, axes, half = case["rows"], case["axes"], case["rotary"] // 2
    i = np.arange(rows)
    if rows <= 16:  # text after images: one position for all axes, another for each row
        positions = np.repeat((1000 + 977 * i)[None], axes, 0)
    else:  # frames of 24 x 32 patches
        positions = np.stack([40 + i // 768, 40 + i // 32 % 24, 40 + i % 32])[:axes]
    j = np.arange(half)
    if case["mixed"]:  # axes in turn, the rest by the first
        pair_axis = np.where(j < half // axes * axes, j % axes, 0)
    else:  # one section after another
        pair_axis = np.minimum(j * axes // half, axes - 1)
    return positions.astype(np.uint32), pair_axis.astype(np.uint8)


def _tensors(case, seed, batch):
    """The case's device arrays, from the seed alone: the pool's pages and the new rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, layers = DTYPES[case["dtype"]], case.get("layers", 1)
    f, qf = case["kv_heads"] * case["head_dim"], case["q_heads"] * case["head_dim"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, dtype=dt, device="cuda")

    t = {"keys": randn(layers, batch.blocks * PAGE, f), "values": randn(layers, batch.blocks * PAGE, f)}
    if case["op"] != "compact":
        rows = len(batch.positions)
        t["k"], t["v"], t["q"] = randn(rows, f), randn(rows, f), randn(rows, qf)
        t["gate"] = randn(rows, qf) if case["gated"] and case["op"] != "rotate" else None
    return t


def _device(a):
    return torch.from_numpy(a.astype(np.int64)).cuda()


def prepare(case, seed):
    batch = _Batch(case, seed)
    t = _tensors(case, seed, batch)
    s = {"case": case, "batch": batch, "scale": 1.0 / math.sqrt(case["head_dim"]), **t}
    if case["op"] != "compact":
        s["out"] = torch.empty_like(t["q"])
    if own:
        from chibillm_amd import ckv

        s["ctx"] = ckv.Context(0, stream=torch.cuda.current_stream())
        s["pool"] = ckv.Pool(s["ctx"], case.get("layers", 1), batch.blocks, PAGE, case["kv_heads"], case["head_dim"],
                             DTYPES[case["dtype"]], t["keys"], t["values"])
        if case["op"] != "compact":
            s["pool"].upload(batch.flat, batch.offsets, batch.lengths, batch.positions, batch.slots)
        if case["op"] == "rotate":
            s["pool"].upload_axes(batch.axes)
    elif case["op"] == "compact":
        s["source"], s["target"], s["shift"] = (_device(x) for x in (batch.source, batch.target, batch.shift))
    else:  # what the framework's upload puts on the device
        s["table"], s["starts"], s["slots"], s["positions"] = (_device(x) for x in (batch.flat, batch.starts, batch.slots, batch.positions))
        s["counts"] = _device(np.array(batch.counts))
        if case["op"] == "rotate":
            s["axes"], s["pair_axis"] = _device(batch.axes), _device(batch.pair_axis)
    return s


# ---- the plain forms ----

def _turn(x, angle, case):
    """Rows [..., heads * head_dim] in 32 bits, pair j of every head turned by angle[..., j] (64 bits)."""
    d, r = case["head_dim"], case["rotary"]
    y = x.reshape(*x.shape[:-1], -1, d)
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    a, b = y[..., :r // 2], y[..., r // 2:r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., r:]], -1).reshape(x.shape)


def _frequencies(case):
    j = torch.arange(case["rotary"] // 2, dtype=torch.float64, device="cuda")
    return case["theta"] ** (-2.0 * j / case["rotary"])


def _slots_of(s, starts, tokens):
    """Slots of a sequence's tokens [sequences, columns] through the tables that start there."""
    return s["table"][starts[:, None] + tokens // PAGE] * PAGE + tokens % PAGE


def _attend(s, q, slots, hidden):
    """softmax(q . k) v over gathered columns: q [b, h, g, n, d] in 32 bits, slots [b, c], hidden [b, n, c]."""
    c = s["case"]
    b, h, g, n, d = q.shape
    k = s["keys"][0][slots].float().reshape(b, -1, h, d).permute(0, 2, 3, 1).contiguous()
    v = s["values"][0][slots].float().reshape(b, -1, h, d).permute(0, 2, 1, 3).contiguous()
    p = torch.matmul(q.reshape(b, h, g * n, d), k).reshape(b, h, g, n, -1) * s["scale"]
    p = p.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p.reshape(b, h, g * n, -1), v).reshape(b, h, g, n, d)


def _plain_decode(s):
    c, batch = s["case"], s["batch"]
    h, d, w, sinks = c["kv_heads"], c["head_dim"], c["window"], c["sinks"]
    rows = len(batch.counts)
    s["keys"][0][s["slots"]], s["values"][0][s["slots"]] = s["k"], s["v"]
    pos = s["positions"]
    low = (pos + 1 - w).clamp(min=0)  # the window's first token
    first = torch.arange(sinks, device="cuda").expand(rows, -1)
    inside = low[:, None] + torch.arange(min(w, c["high"]), device="cuda")
    tokens = torch.cat([first, inside], 1)
    hidden = torch.cat([first >= low[:, None], inside > pos[:, None]], 1)
    tokens = torch.minimum(tokens, pos[:, None])
    q = s["q"].float().reshape(rows, h, -1, 1, d)
    out = _attend(s, q, _slots_of(s, s["starts"], tokens), hidden[:, None]).reshape(rows, -1)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    s["out"].copy_(out)
    return {"out": s["out"], "keys": s["keys"], "values": s["values"]}


def _plain_prefill(s):
    c, batch = s["case"], s["batch"]
    h, d, w, sinks, prefix = c["kv_heads"], c["head_dim"], c["window"], c["sinks"], c["prefix"]
    b, n = len(batch.counts), max(batch.counts)
    i = torch.arange(n, device="cuda")
    mine = i < s["counts"][:, None]  # [b, n]: rows that are there
    row = (s["counts"].cumsum(0) - s["counts"])[:, None] + torch.minimum(i, s["counts"][:, None] - 1)
    base = max(0, prefix + 1 - w)  # the first row's window begins there
    first, inside = torch.arange(sinks, device="cuda"), torch.arange(base, prefix + n, device="cuda")
    tokens = torch.cat([first, inside])
    pos = prefix + i[:, None]
    hidden = torch.cat([(first >= base).expand(n, -1), (inside > pos) | ((inside <= pos - w) & (inside >= sinks))], 1)
    ends = (prefix + s["counts"])[:, None]
    slots = _slots_of(s, s["starts"], torch.minimum(tokens, ends - 1))
    q = s["q"][row].float().reshape(b, n, h, -1, d).permute(0, 2, 3, 1, 4)
    out = _attend(s, q, slots, hidden.expand(b, -1, -1)).permute(0, 3, 1, 2, 4).reshape(b, n, -1)[mine]
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    s["out"].copy_(out)
    return {"out": s["out"]}


def _plain_rotate(s):
    c = s["case"]
    angle = s["axes"][s["pair_axis"]].t().double() * _frequencies(c)  # [rows, pairs]
    s["out"].copy_(_turn(s["q"].float(), angle, c))
    s["keys"][0][s["slots"]] = _turn(s["k"].float(), angle, c).to(s["keys"].dtype)
    s["values"][0][s["slots"]] = s["v"]
    return {"out": s["out"], "keys": s["keys"], "values": s["values"]}


def _plain_compact(s):
    c = s["case"]
    turned = _turn(s["keys"][:, s["source"]].float(), s["shift"][:, None].double() * _frequencies(c), c)
    s["keys"][:, s["target"]] = turned.to(s["keys"].dtype)
    s["values"][:, s["target"]] = s["values"][:, s["source"]]
    return {"keys": s["keys"], "values": s["values"]}


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"decode": _plain_decode, "prefill": _plain_prefill, "rotate": _plain_rotate, "compact": _plain_compact}[op](s)
    pool, batch = s["pool"], s["batch"]
    if op == "compact":
        pool.compact(batch.source, batch.target, [x.size for x in batch.kept], batch.shift, c["theta"], c["rotary"])
        return {"keys": s["keys"], "values": s["values"]}
    if op == "prefill":
        pool.attention_window(0, s["q"], c["q_heads"], s["scale"], c["window"], s["out"], sinks=c["sinks"], gate=s["gate"])
        return {"out": s["out"]}
    if op == "decode":
        pool.append_decode_window(0, s["k"], s["v"], s["q"], c["q_heads"], s["scale"], c["window"], s["out"], sinks=c["sinks"], gate=s["gate"])
    else:
        pool.rope_axes_append(0, s["q"], s["out"], c["q_heads"], s["k"], s["v"], c["theta"], batch.pair_axis, c["rotary"])
    return {"out": s["out"], "keys": s["keys"], "values": s["values"]}


def work(case):
    """Bytes read and written once, and the products of q.k and p.v that the mask leaves."""
    size = 4 if case["dtype"] == "f32" else 2
    f, qf = case["kv_heads"] * case["head_dim"], case["q_heads"] * case["head_dim"]
    if case["op"] == "compact":
        moved = 0
        for n in _spread(case["sequences"], case["low"], case["high"]):
            kept = _kept(case, n)
            moved += kept.size - (0 if case["fresh"] else int((kept == np.arange(kept.size)).sum()))
        return {"bytes": 4.0 * case["layers"] * moved * f * size, "flops": 0.0}
    if case["op"] == "rotate":
        return {"bytes": float(case["rows"] * (4 * f + 2 * qf) * size), "flops": 0.0}
    w, sinks = case["window"], case["sinks"]

    def seen(p):  # keys that a row at position p attends
        low = max(0, p + 1 - w)
        return p + 1 - low + min(sinks, low)

    gate = 1 if case["gated"] else 0
    if case["op"] == "decode":
        spans = _spread(case["rows"], case["low"], case["high"])
        pairs = sum(seen(n - 1) for n in spans)
        moved = (pairs - len(spans)) * 2 * f + len(spans) * 4 * f + len(spans) * qf * (2 + gate)
    else:
        prefix, counts = case["prefix"], _spread(case["sequences"], case["rows_low"], case["rows_high"])
        pairs = sum(seen(prefix + i) for n in counts for i in range(n))
        held = sum(n - 1 + seen(prefix) for n in counts)
        moved = held * 2 * f + sum(counts) * qf * (2 + gate)
    return {"bytes": float(moved * size), "flops": 4.0 * pairs * qf}


# ---- the same calls in 64 bits ----

def _rotated(x, angle, case):
    """Each head's pairs as complex numbers, turned."""
    d, r = case["head_dim"], case["rotary"]
    y = x.double().unflatten(-1, (-1, d)).clone()
    z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * torch.polar(torch.ones_like(angle), angle).unsqueeze(-2)
    y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y.flatten(-2)


def exact(case, seed):
    batch = _Batch(case, seed)
    t = _tensors(case, seed, batch)
    inverse = torch.exp(-2.0 * math.log(case["theta"]) * torch.arange(case["rotary"] // 2, dtype=torch.float64, device="cuda") / case["rotary"])
    if case["op"] == "compact":
        source, target, shift = (_device(x) for x in (batch.source, batch.target, batch.shift))
        keys, values = t["keys"].double(), t["values"].double()
        keys[:, target] = _rotated(t["keys"][:, source], shift.double()[:, None] * inverse, case)
        values[:, target] = t["values"][:, source].double()
        return {"keys": keys, "values": values}
    keys, values = t["keys"].double(), t["values"].double()
    slots = _device(batch.slots)
    if case["op"] == "rotate":
        at = _device(batch.axes).double()[_device(batch.pair_axis)]
        angle = torch.einsum("jr,j->rj", at, inverse)
        keys[0, slots], values[0, slots] = _rotated(t["k"], angle, case), t["v"].double()
        return {"out": _rotated(t["q"], angle, case), "keys": keys, "values": values}
    if case["op"] == "decode":
        keys[0, slots], values[0, slots] = t["k"].double(), t["v"].double()
    h, d, w, sinks = case["kv_heads"], case["head_dim"], case["window"], case["sinks"]
    out, row = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda"), 0
    for table, first, count in zip(batch.tables, batch.first, batch.counts):
        p = np.arange(first + count)
        p = p[(p > first - w) | (p < sinks)]  # what the first row or a later one attends
        at = _device(batch._slot(table, p))
        p = torch.from_numpy(p).cuda()
        position = torch.arange(first, first + count, device="cuda")[:, None]
        seen = (p <= position) & ((p > position - w) | (p < sinks))
        for head in range(case["q_heads"]):
            of = slice(head // (case["q_heads"] // h) * d, (head // (case["q_heads"] // h) + 1) * d)
            q = t["q"][row:row + count, head * d:(head + 1) * d].double()
            e = torch.where(seen, q @ keys[0, at, of].t().contiguous() / math.sqrt(d), -math.inf).softmax(-1)
            out[row:row + count, head * d:(head + 1) * d] = e @ values[0, at, of]
        row += count
    if t["gate"] is not None:
        out *= torch.sigmoid(t["gate"].double())
    return {"out": out, "keys": keys, "values": values} if case["op"] == "decode" else {"out": out}
