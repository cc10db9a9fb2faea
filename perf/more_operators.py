"""Operators of a serving program whose cache is held in 4 bits, as calls to measure.

Such a program keeps keys and values as 4-bit floats (1 sign, 2 exponent and 1 mantissa
bit) with one power of two for each 32 features of a head. New rows are rotated by their
positions (neighbouring or halved pairs, part of the head, frequencies scaled for long
contexts) and appended in one call; whole prompts attend to their own rows, as the cache
holds them; later chunks and decode rows attend to the cache. The cases are single calls of
these on a paged pool whose pages are scattered. Values are N(0, 1) from the seed.

`own` false computes a call in elementary torch operations, true calls `chibillm_amd.ckv`;
`exact` answers in 64 bits.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LOWEST = {"bf16": -100, "f16": -23, "f32": -100}  # the smallest scale's exponent, by the rows' type

# Heads of one attention layer. "narrow": the KV shape of the benchmark's model. "wide": a
# layer with an output gate, 256-wide heads and rotary on a quarter of the head. "slim": a
# small model's 64-wide heads.
NARROW = {"kv_heads": 8, "q_heads": 16, "head_dim": 128, "rotary": 128, "theta": 1e6, "gated": False}
WIDE = {"kv_heads": 2, "q_heads": 8, "head_dim": 256, "rotary": 64, "theta": 1e7, "gated": True}
SLIM = {"kv_heads": 4, "q_heads": 4, "head_dim": 64, "rotary": 64, "theta": 1e4, "gated": False}

# Scaling of the frequencies: positions divided by a factor; long wavelengths alone
# divided, with a blend between two bands; the same by pair index, with a magnitude.
SCALINGS = {
    "none": {},
    "linear": {"factor": 4.0},
    "bands": {"factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
    "yarn": {"factor": 4.0, "low": 1.0, "high": 32.0, "original": 32768},
}


def _case(op, heads, **more):
    return {"op": op, **heads, "dtype": "bf16", **more}


def listed():
    return [
        # a decode step of a few chats on a 16-bit pool, frequencies scaled by bands
        dict(_case("rotate", NARROW, rows=7, layout="halves", scaling="bands"), name="rotate decode rows"),
        # a long prompt of a layer with wide heads, neighbouring pairs, a quarter of the head
        dict(_case("rotate", WIDE, rows=4999, layout="pairs", scaling="yarn", dtype="f16"), name="rotate prompt"),
        # new prompts into the 4-bit cache, rows as it holds them returned for their attention
        dict(_case("append", NARROW, rows=4096, layout="halves", scaling="yarn"), name="fp4 append prompts"),
        # an odd chunk of neighbouring pairs, f32 rows
        dict(_case("append", SLIM, rows=333, layout="pairs", scaling="linear", dtype="f32"), name="fp4 append chunk"),
        # the smallest call: one decode step of four chats, from unrotated rows
        dict(_case("step", NARROW, rows=4, low=60, high=1900, layout="halves", scaling="yarn"), name="fp4 step 4 rows"),
        # an ordinary serving batch
        dict(_case("decode", NARROW, rows=48, low=900, high=12000), name="fp4 decode 48 rows"),
        # the largest batch, bound by the cache's bytes
        dict(_case("decode", NARROW, rows=128, low=3000, high=8000), name="fp4 decode 128 rows"),
        # a gated layer with wide heads
        dict(_case("decode", WIDE, rows=24, low=200, high=9000, dtype="f16"), name="fp4 decode wide heads"),
        # the middle of a long prompt: one sequence's next chunk over the 4-bit cache
        dict(_case("chunk", NARROW, sequences=1, rows_low=512, rows_high=512, prefix=6000), name="fp4 chunk"),
        # new prompts of mixed lengths packed together, attended from their rows
        dict(_case("prompt", NARROW, sequences=9, rows_low=17, rows_high=900, dtype="f16"), name="prompt packed"),
        # two long documents
        dict(_case("prompt", NARROW, sequences=2, rows_low=6000, rows_high=8192), name="prompt long"),
        # rows in the storage type of the reference engine
        dict(_case("prompt", SLIM, sequences=5, rows_low=1, rows_high=700, dtype="f32"), name="prompt f32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges; none costs more than the largest listed one."""
    op = rng.choice(["rotate", "append", "append", "step", "decode", "decode", "decode", "chunk", "chunk", "prompt", "prompt", "prompt"])
    heads = dict(rng.choice([NARROW, NARROW, WIDE, SLIM]))
    if heads["head_dim"] != 128:  # the same layer at other head counts of its kind
        heads["kv_heads"] = rng.choice([1, 2, 4])
        heads["q_heads"] = heads["kv_heads"] * rng.choice([1, 2, 4, 8])
    heads["gated"] = heads["gated"] and rng.random() < 0.7
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    turn = {"layout": rng.choice(["halves", "pairs"]), "scaling": rng.choice(list(SCALINGS))}
    if op in ("rotate", "append"):
        return _case(op, heads, rows=_log(rng, 1, 4096), dtype=dtype, **turn)
    if op in ("step", "decode"):
        rows = _log(rng, 1, 128)
        high = _log(rng, 40, max(64, min(16000, 700_000 // rows)))
        more = turn if op == "step" else {}
        return _case(op, heads, rows=rows, low=max(1, int(high * rng.uniform(0.05, 1.0))), high=high, dtype=dtype, **more)
    high = _log(rng, 9, 4096 if op == "prompt" else 1024)
    if op == "chunk":
        sequences = _log(rng, 1, 8)
        case = _case(op, heads, sequences=sequences, rows_low=max(2, int(high * rng.uniform(0.1, 1.0))), rows_high=high,
                     prefix=_log(rng, 3, 6000), dtype=dtype)
    else:
        sequences = _log(rng, 1, max(1, min(24, 12_000 // high)))
        case = _case(op, heads, sequences=sequences, rows_low=max(1, int(high * rng.uniform(0.02, 1.0))), rows_high=high, dtype=dtype)
    while work(case)["flops"] > (1e11 if dtype == "f32" else 3e11):
        case["sequences"] = (case["sequences"] + 1) // 2
        case["q_heads"] = max(case["kv_heads"], case["q_heads"] // 2)
    return case


# ---- shapes of a case (the same for every seed) ----

def _spread(n, low, high):
    """n lengths spread evenly over [low, high], in a mixed order."""
    order = np.random.RandomState(n).permutation(n)
    return [int(x) for x in np.round(np.linspace(low, high, n))[order]] if n > 1 else [high]


class _Batch:
    """Tables, positions and slots of a case's rows, over pages in an order drawn from the seed."""

    def __init__(self, case, seed):
        op = case["op"]
        if op in ("rotate", "append"):
            counts, first = [case["rows"]], [0 if case["rows"] > 16 else 20_001]  # far on in a chat
        elif op in ("step", "decode"):
            spans = _spread(case["rows"], case["low"], case["high"])
            counts, first = [1] * len(spans), [n - 1 for n in spans]
        else:
            counts = _spread(case["sequences"], case["rows_low"], case["rows_high"])
            first = [case.get("prefix", 0)] * len(counts)
        self.counts, self.first = counts, first
        pages = [-(-(f + c) // PAGE) for f, c in zip(first, counts)]
        self.blocks = sum(pages) + 5
        order = np.random.RandomState(seed % (1 << 32)).permutation(self.blocks).astype(np.uint32)
        self.flat = order[:sum(pages)]
        self.starts = np.concatenate([[0], np.cumsum(pages)[:-1]])
        seq = np.repeat(np.arange(len(counts)), counts)
        self.positions = np.concatenate([np.arange(f, f + c) for f, c in zip(first, counts)]).astype(np.uint32)
        self.offsets = self.starts[seq].astype(np.uint32)
        self.lengths = np.array(pages, np.uint32)[seq]
        page = self.flat[self.offsets + self.positions // PAGE]
        self.slots = (page.astype(np.uint64) * PAGE + self.positions % PAGE).astype(np.uint32)

    def slots_of(self, i):
        """Slots of sequence i's tokens, its last row's among them."""
        p = np.arange(self.first[i] + self.counts[i])
        return self.flat[self.starts[i] + p // PAGE].astype(np.int64) * PAGE + p % PAGE


FP4 = ("append", "step", "decode", "chunk")  # the operators on a pool held in 4 bits


def _tensors(case, seed, batch):
    """The case's device arrays, from the seed alone: the new rows, and rows for the pool's slots."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]
    f, qf, rows = case["kv_heads"] * case["head_dim"], case["q_heads"] * case["head_dim"], len(batch.positions)

    def randn(*shape):
        return torch.randn(*shape, generator=g, dtype=dt, device="cuda")

    t = {"k": randn(rows, f), "v": randn(rows, f), "q": randn(rows, qf)}
    t["gate"] = randn(rows, qf) if case["gated"] and op not in ("rotate", "append") else None
    if op in ("rotate", "step", "decode", "chunk"):
        t["keys"], t["values"] = randn(batch.blocks * PAGE, f), randn(batch.blocks * PAGE, f)
    return t


def _device(a):
    return torch.from_numpy(a.astype(np.int64)).cuda()


def _magnitude(case):
    return 0.1 * math.log(SCALINGS["yarn"]["factor"]) + 1.0 if case["scaling"] == "yarn" else 1.0


def prepare(case, seed):
    batch = _Batch(case, seed)
    t, op = _tensors(case, seed, batch), case["op"]
    filled = [t.pop("keys", None), t.pop("values", None)]
    s = {"case": case, "batch": batch, "scale": 1.0 / math.sqrt(case["head_dim"]), **t, "out": torch.empty_like(t["q"])}
    if op in ("append", "step"):
        s["held_k"], s["held_v"] = torch.empty_like(t["k"]), torch.empty_like(t["v"])
    if op == "rotate":
        s["keys"], s["values"] = filled
    if own:
        from chibillm_amd import ckv

        s["ctx"] = ckv.Context(0, stream=torch.cuda.current_stream())
        geometry = (s["ctx"], 1, batch.blocks, PAGE, case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]])
        s["pool"] = pool = ckv.Pool(*geometry, *(filled if op == "rotate" else ()), fp4=op in FP4)
        if op in ("step", "decode", "chunk"):
            slots = np.arange(batch.blocks * PAGE)
            pool.upload(np.arange(batch.blocks), slots // PAGE, np.ones(slots.size), slots % PAGE, slots)
            pool.append(0, *filled)
        pool.upload(batch.flat, batch.offsets, batch.lengths, batch.positions, batch.slots)
        if "scaling" in case:
            s["rotation"] = ckv.Rotation(case["theta"], case["rotary"], case["layout"], case["scaling"], **SCALINGS[case["scaling"]])
        return s
    # what the framework's upload puts on the device
    s["table"], s["starts"], s["slots"], s["positions"] = (_device(x) for x in (batch.flat, batch.starts, batch.slots, batch.positions))
    s["counts"], s["first"] = _device(np.array(batch.counts)), _device(np.array(batch.first))
    if "scaling" in case:
        s["inverse"] = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
    if op in FP4:
        s["levels"] = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
        f = case["kv_heads"] * case["head_dim"]
        for name, x in zip(("keys", "values"), filled):
            codes = torch.zeros(batch.blocks * PAGE, f // 2, dtype=torch.uint8, device="cuda")
            scales = torch.zeros(batch.blocks * PAGE, f // 32, dtype=torch.uint8, device="cuda")
            if x is not None:
                for at in range(0, len(x), 1 << 15):
                    codes[at:at + (1 << 15)], scales[at:at + (1 << 15)] = _quantised(x[at:at + (1 << 15)].float(), case)
            s[name] = (codes, scales)
    return s


# ---- the plain forms ----

def _frequencies(case):
    """Radians by which a step of one position turns each pair."""
    r, theta = case["rotary"], case["theta"]
    f = [theta ** (-2.0 * j / r) for j in range(r // 2)]
    w = SCALINGS[case["scaling"]]
    if case["scaling"] == "linear":
        return [x / w["factor"] for x in f]
    if case["scaling"] == "bands":
        turns = [w["original"] * x / (2 * math.pi) for x in f]  # in the original context
        keep = [min(1.0, max(0.0, (t - w["low"]) / (w["high"] - w["low"]))) for t in turns]
        return [x * (k + (1 - k) / w["factor"]) for x, k in zip(f, keep)]
    if case["scaling"] == "yarn":
        def pair(turns):  # the pair that makes so many in the original context
            return r * math.log(w["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(0, math.floor(pair(w["high"]))), min(r - 1, math.ceil(pair(w["low"])))
        ramp = [min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(r // 2)]
        return [x * (1 - k) + x / w["factor"] * k for x, k in zip(f, ramp)]
    return f


def _turned(x, s, wide=False):
    """Rows rotated by their positions: in 32 bits, or in 64, which decide at the levels' borders."""
    c = s["case"]
    d, r = c["head_dim"], c["rotary"]
    angle = s["positions"].double()[:, None] * s["inverse"]
    cos, sin = angle.cos() * _magnitude(c), angle.sin() * _magnitude(c)
    y = x.double() if wide else x.float()
    cos, sin = cos.to(y.dtype)[:, None], sin.to(y.dtype)[:, None]
    y = y.reshape(len(x), -1, d)
    if c["layout"] == "halves":
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., :r:2], y[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., r:]], -1).reshape(x.shape)


def _power(exponent):
    """2^exponent, exactly."""
    return (exponent + 127 << 23).view(torch.float32)


def _quantised(x, case):
    """(packed codes, scale bytes) of rows: each 32 features over 2^e, with e from their largest, to the nearest level."""
    y = x.reshape(len(x), -1, 32)
    exponent = torch.frexp(y.abs().amax(-1, keepdim=True)).exponent.int() - 3  # its binade, two below
    exponent = exponent.clamp(min=LOWEST[case["dtype"]])
    y = y * _power(-exponent)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte()
            + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5).byte())  # ties to the even code
    code = (code + 8 * torch.signbit(y).byte()).reshape(len(x), -1)
    return code[:, ::2] | code[:, 1::2] << 4, (exponent.squeeze(-1) + 127).byte()


def _held(codes, scales, s):
    """The values that codes and scales stand for, in 32 bits."""
    x = torch.stack([s["levels"][(codes & 15).int()], s["levels"][(codes >> 4).int()]], -1).flatten(-2)
    return (x.reshape(*scales.shape, 32) * _power(scales.int() - 127)[..., None]).flatten(-2)


def _attend(s, q, k, v, hidden):
    """softmax(q . k) v: q [b, h, g, n, d], k and v [b, c, h * d], all in 32 bits, hidden [b, n, c]."""
    b, h, g, n, d = q.shape
    k = k.reshape(b, -1, h, d).permute(0, 2, 3, 1).contiguous()
    v = v.reshape(b, -1, h, d).permute(0, 2, 1, 3).contiguous()
    p = torch.matmul(q.reshape(b, h, g * n, d), k).reshape(b, h, g, n, -1) * s["scale"]
    p = p.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p.reshape(b, h, g * n, -1), v).reshape(b, h, g, n, d)


def _store(s, out):
    """The attention's rows, gated, rounded once."""
    s["out"].copy_(out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].float())))
    return s["out"]


def _put(s, k, v):
    """Rows into the 4-bit cache, and into the rows it then holds."""
    for name, x in (("k", k), ("v", v)):
        codes, scales = _quantised(x, s["case"])
        cache = s["keys" if name == "k" else "values"]
        cache[0][s["slots"]], cache[1][s["slots"]] = codes, scales
        s["held_" + name].copy_(_held(codes, scales, s))


def _plain_rotate(s):
    s["out"].copy_(_turned(s["q"], s))
    s["keys"][s["slots"]] = _turned(s["k"], s).to(s["keys"].dtype)
    s["values"][s["slots"]] = s["v"]
    return {"out": s["out"], "keys": s["keys"], "values": s["values"]}


def _plain_append(s):
    s["out"].copy_(_turned(s["q"], s))
    _put(s, _turned(s["k"], s, wide=True), s["v"].float())
    return {"out": s["out"], "keys": s["held_k"], "values": s["held_v"]}


def _cached(s):
    """Every row of the batch at once over its sequence's cached tokens."""
    c = s["case"]
    b, n, h, d = len(s["counts"]), int(max(s["batch"].counts)), c["kv_heads"], c["head_dim"]
    i = torch.arange(n, device="cuda")
    mine = i < s["counts"][:, None]  # [b, n]: rows that are there
    row = (s["counts"].cumsum(0) - s["counts"])[:, None] + torch.minimum(i, s["counts"][:, None] - 1)
    ends = (s["first"] + s["counts"])[:, None]
    tokens = torch.arange(max(f + m for f, m in zip(s["batch"].first, s["batch"].counts)), device="cuda")
    hidden = tokens > (s["first"][:, None] + i)[..., None]
    at = torch.minimum(tokens, ends - 1)
    slots = s["table"][s["starts"][:, None] + at // PAGE] * PAGE + at % PAGE
    k, v = (_held(cache[0][slots], cache[1][slots], s) for cache in (s["keys"], s["values"]))
    q = s["turned"][row].float().reshape(b, n, h, -1, d).permute(0, 2, 3, 1, 4)
    return _attend(s, q, k, v, hidden).permute(0, 3, 1, 2, 4).reshape(b, n, -1)[mine]


def _plain_step(s):
    s["turned"] = _turned(s["q"], s)
    _put(s, _turned(s["k"], s, wide=True), s["v"].float())
    return {"out": _store(s, _cached(s)), "keys": s["held_k"], "values": s["held_v"]}


def _plain_cached(s):
    s["turned"] = s["q"]
    return {"out": _store(s, _cached(s))}


def _plain_prompt(s):
    c = s["case"]
    b, n, h, d = len(s["counts"]), max(s["batch"].counts), c["kv_heads"], c["head_dim"]
    i = torch.arange(n, device="cuda")
    mine = i < s["counts"][:, None]
    row = (s["counts"].cumsum(0) - s["counts"])[:, None] + torch.minimum(i, s["counts"][:, None] - 1)
    q = s["q"][row].float().reshape(b, n, h, -1, d).permute(0, 2, 3, 1, 4)
    out = _attend(s, q, s["k"][row].float(), s["v"][row].float(), (i > i[:, None]).expand(b, -1, -1))
    return {"out": _store(s, out.permute(0, 3, 1, 2, 4).reshape(b, n, -1)[mine])}


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"rotate": _plain_rotate, "append": _plain_append, "step": _plain_step, "decode": _plain_cached,
                "chunk": _plain_cached, "prompt": _plain_prompt}[op](s)
    pool = s["pool"]
    if op == "rotate":
        pool.rotate_append(0, s["rotation"], s["q"], s["out"], c["q_heads"], s["k"], s["v"])
        return {"out": s["out"], "keys": s["keys"], "values": s["values"]}
    if op == "append":
        pool.rotate_append(0, s["rotation"], s["q"], s["out"], c["q_heads"], s["k"], s["v"], held_keys=s["held_k"], held_values=s["held_v"])
        return {"out": s["out"], "keys": s["held_k"], "values": s["held_v"]}
    if op == "step":
        pool.rotate_append_decode(0, s["rotation"], s["k"], s["v"], s["q"], c["q_heads"], s["scale"], s["out"], gate=s["gate"],
                                  held_keys=s["held_k"], held_values=s["held_v"])
        return {"out": s["out"], "keys": s["held_k"], "values": s["held_v"]}
    if op == "prompt":
        pool.prompt_attention(s["q"], s["k"], s["v"], c["q_heads"], s["scale"], s["out"], gate=s["gate"])
    elif s["gate"] is not None:
        pool.attention_gated(0, s["q"], c["q_heads"], s["scale"], s["gate"], s["out"])
    else:
        pool.attention(0, s["q"], c["q_heads"], s["scale"], s["out"])
    return {"out": s["out"]}


def work(case):
    """Bytes read and written once, and the products of q.k and p.v that the mask leaves."""
    size = 4 if case["dtype"] == "f32" else 2
    f, qf, op = case["kv_heads"] * case["head_dim"], case["q_heads"] * case["head_dim"], case["op"]
    token = f + f / 16  # bytes of a token's keys and values in 4 bits, scales among them
    gate = 1 if case["gated"] else 0
    if op == "rotate":
        return {"bytes": float(case["rows"] * (4 * f + 2 * qf) * size), "flops": 0.0}
    if op == "append":
        return {"bytes": float(case["rows"] * ((4 * f + 2 * qf) * size + token)), "flops": 0.0}
    if op in ("step", "decode"):
        spans = _spread(case["rows"], case["low"], case["high"])
        pairs = sum(spans)
        moved = pairs * token + len(spans) * (qf * (2 + gate) + (4 * f if op == "step" else 0)) * size
    else:
        prefix, counts = case.get("prefix", 0), _spread(case["sequences"], case["rows_low"], case["rows_high"])
        pairs = sum(n * prefix + n * (n + 1) // 2 for n in counts)
        moved = sum((n + prefix) * token if op == "chunk" else n * 2 * f * size for n in counts) + sum(counts) * qf * (2 + gate) * size
    return {"bytes": float(moved), "flops": 4.0 * pairs * qf}


# ---- the same calls in 64 bits ----

def _steps(case):
    """Radians per position of each pair, in 64 bits on the device."""
    r = case["rotary"]
    j = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(-2.0 * j / r * math.log(case["theta"]))
    w = SCALINGS[case["scaling"]]
    if case["scaling"] == "linear":
        return f / w["factor"]
    if case["scaling"] == "bands":
        length = 2 * math.pi / f
        blend = (w["original"] / length - w["low"]) / (w["high"] - w["low"])
        between = (1 - blend) * f / w["factor"] + blend * f
        return torch.where(length < w["original"] / w["high"], f, torch.where(length > w["original"] / w["low"], f / w["factor"], between))
    if case["scaling"] == "yarn":
        first = math.floor(r / 2 * math.log(w["original"] / (2 * math.pi * w["high"]), case["theta"]))
        last = math.ceil(r / 2 * math.log(w["original"] / (2 * math.pi * w["low"]), case["theta"]))
        first, last = max(first, 0), min(last, r - 1)
        mix = ((j - first) / max(last - first, 0.001)).clamp(0, 1)
        return f / w["factor"] * mix + f * (1 - mix)
    return f


def _rotated(x, positions, case):
    """Each head's pairs as complex numbers, turned and lengthened."""
    d, r = case["head_dim"], case["rotary"]
    y = x.double().unflatten(-1, (-1, d)).clone()
    angle = positions.double()[:, None] * _steps(case)
    turn = torch.polar(torch.full_like(angle, _magnitude(case)), angle).unsqueeze(-2)
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "halves" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y.flatten(-2)


def _rounded(x, case):
    """Rows as a 4-bit cache holds them: multiples of a half, one or two of their scale, at most six."""
    y = x.double().unflatten(-1, (-1, 32))
    largest = y.abs().amax(-1, keepdim=True)
    power = torch.floor(torch.log2(largest))
    power = power + (torch.exp2(power + 1) <= largest).double() - (torch.exp2(power) > largest).double() - 2  # the logarithm is rounded
    unit = torch.exp2(power.clamp(min=LOWEST[case["dtype"]]))
    a = (y / unit).abs()
    grain = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.copysign((torch.round(a / grain) * grain).clamp(max=6), y) * unit).flatten(-2)


def exact(case, seed):
    batch, op = _Batch(case, seed), case["op"]
    t = _tensors(case, seed, batch)
    slots, positions = _device(batch.slots), _device(batch.positions)
    if op == "rotate":
        keys, values = t["keys"].double(), t["values"].double()
        keys[slots], values[slots] = _rotated(t["k"], positions, case), t["v"].double()
        return {"out": _rotated(t["q"], positions, case), "keys": keys, "values": values}
    if op in ("append", "step"):
        q, held_k, held_v = _rotated(t["q"], positions, case), _rounded(_rotated(t["k"], positions, case), case), _rounded(t["v"], case)
        if op == "append":
            return {"out": q, "keys": held_k, "values": held_v}
    else:
        q = t["q"].double()
    h, d, row = case["kv_heads"], case["head_dim"], 0
    group, out = case["q_heads"] // h, torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    for i, (first, count) in enumerate(zip(batch.first, batch.counts)):
        if op == "prompt":
            k, v = t["k"][row:row + count].double(), t["v"][row:row + count].double()
        else:
            at = torch.from_numpy(batch.slots_of(i)).cuda()
            k, v = _rounded(t["keys"][at], case), _rounded(t["values"][at], case)
        if op == "step":
            k[-1], v[-1] = held_k[row], held_v[row]
        seen = torch.arange(len(k), device="cuda") <= torch.arange(first, first + count, device="cuda")[:, None]
        for head in range(case["q_heads"]):
            of = slice(head // group * d, (head // group + 1) * d)
            e = torch.where(seen, q[row:row + count, head * d:(head + 1) * d] @ k[:, of].t().contiguous() / math.sqrt(d), -math.inf).softmax(-1)
            out[row:row + count, head * d:(head + 1) * d] = e @ v[:, of].contiguous()
        row += count
    if t["gate"] is not None:
        out *= torch.sigmoid(t["gate"].double())
    return {"out": out, "keys": held_k, "values": held_v} if op == "step" else {"out": out}
