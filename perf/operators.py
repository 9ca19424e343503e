"""Cases of the token-memory operators: rotary positions over time, height and width, the norm of queries and keys in the same
pass, and a memory bank held in 4 bits (append, attention read, eviction by the attention weight its slots have received).

`run` with `own = False` computes every operator in its plain form (elementary torch operations, fp32, angles in fp64, rounded once
at the end); with `own = True` it makes the calls of mivos_amd.ops.  Both work on the tensors that `prepare` makes.

The 4-bit format, shared by both forms: a row of D channels is D/32 blocks; a block is one power of two 2^(byte - 127), the
smallest with max |x| <= 6 * 2^e (e within [-120, 125]; byte 255 = the block holds an infinity or a NaN and stands for NaN), and 32
codes of sign, two exponent bits and one mantissa bit (+-{0, 0.5, 1, 1.5, 2, 3, 4, 6}), rounded to nearest, ties to the even code.
Codes are packed two to a byte, the even channel in the low half.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of each of 8 streams, no norm, neighbouring channels paired, far along the time axis: a latency call
        dict(name="rotary token", op="rotary", grad=False, dtype="fp16", batch=8, tokens=1, q_heads=8, k_heads=2, dim=64,
             axes="8,12,12", interleaved=True, shared=False, base=10000.0, width=54, height=30, time0=70000),
        # training on three clips of one 480p frame (30 x 54 tokens) with heads of 80 channels in fp32: gradients of q and k
        dict(name="rotary frames grad", op="rotary", grad=True, dtype="fp32", batch=3, tokens=1620, q_heads=5, k_heads=5, dim=80,
             axes="8,16,16", interleaved=False, shared=False, base=10000.0, width=54, height=30, time0=0),
        # the tokens of 20 bank frames at 480p, grouped heads, q and k as slices of one projection
        dict(name="norm rotary clip", op="norm_rotary", grad=False, dtype="bf16", batch=1, tokens=32400, q_heads=16, k_heads=4, dim=128,
             axes="16,24,24", interleaved=False, shared=False, base=10000.0, width=54, height=30, time0=0),
        # the same layer's backward pass on two clips of five frames: gradients of q, k and both norm weights
        dict(name="norm rotary clip grad", op="norm_rotary", grad=True, dtype="bf16", batch=2, tokens=8100, q_heads=16, k_heads=4, dim=128,
             axes="16,24,24", interleaved=False, shared=False, base=10000.0, width=54, height=30, time0=0),
        # one new token of each of 16 streams into the bank: a latency call
        dict(name="append tokens", op="append", dtype="bf16", batch=16, heads=8, key_dim=128, value_dim=128, tokens=1, slots=4096, ragged=True),
        # one 1080p frame (68 x 120 positions) of three objects in the layout of the space-time memory: key 128, value 512
        dict(name="append frame 1080p", op="append", dtype="fp32", batch=3, heads=1, key_dim=128, value_dim=512, tokens=8160, slots=24480, ragged=False),
        # one token against a short bank: a latency call
        dict(name="read token", op="read", dtype="fp16", batch=1, q_heads=8, heads=2, key_dim=64, value_dim=64, tokens=1, slots=1024,
             fill=1000, ragged=False, causal=False, weigh=False),
        # one token of each of four streams against long banks of different lengths, weights gathered for the next eviction
        dict(name="read token long", op="read", dtype="bf16", batch=4, q_heads=32, heads=8, key_dim=128, value_dim=128, tokens=1, slots=131072,
             fill=131000, ragged=True, causal=False, weigh=True),
        # one 480p frame of two objects against a bank of 20 frames, key 128 and value 512, weights gathered
        dict(name="read frame 480p", op="read", dtype="fp32", batch=2, q_heads=1, heads=1, key_dim=128, value_dim=512, tokens=1620, slots=32400,
             fill=32400, ragged=False, causal=False, weigh=True),
        # a prompt of an odd length behind what the bank already holds, causal, four query heads on each bank head
        dict(name="read prompt causal", op="read", dtype="bf16", batch=3, q_heads=16, heads=4, key_dim=128, value_dim=128, tokens=1021, slots=16384,
             fill=16300, ragged=True, causal=True, weigh=False),
        # one object's bank of 13 frames at 480p brought down to 10, the first frame and the newest one kept
        dict(name="evict frames", op="evict", dtype="bf16", batch=1, heads=1, key_dim=128, value_dim=512, slots=21060, keep=16200, first=1620,
             recent=1620, ragged=False),
        # four streams' banks of eight heads brought down to three quarters
        dict(name="evict streams", op="evict", dtype="bf16", batch=4, heads=8, key_dim=128, value_dim=128, slots=32768, keep=24576, first=4,
             recent=512, ragged=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rotary", "norm_rotary", "append", "read", "read", "evict"))
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    if op in ("rotary", "norm_rotary"):
        dim = rng.choice((32, 64, 72, 80, 96, 128, 256))
        pairs = dim // 2 if rng.random() < 0.7 else rng.randint(3, dim // 2)
        a = rng.randint(1, pairs - 2)
        b = rng.randint(1, pairs - a - 1)
        k_heads = rng.choice((1, 2, 3, 4, 8))
        q_heads = k_heads * rng.choice((1, 2, 4))
        batch = rng.randint(1, 8)
        most = 32400 * 20 * 80 // (batch * (q_heads + k_heads) * dim)
        return dict(op=op, grad=rng.random() < 0.5, dtype=dtype, batch=batch, tokens=_log(rng, 1, min(most, 40000)), q_heads=q_heads, k_heads=k_heads,
                    dim=dim, axes="%d,%d,%d" % (a, b, pairs - a - b), interleaved=rng.random() < 0.5, shared=rng.random() < 0.3,
                    base=rng.choice((100.0, 10000.0, 500000.0)), width=rng.randint(1, 120), height=rng.randint(1, 68),
                    time0=rng.choice((0, 0, _log(rng, 10, 1000000))))
    key_dim, value_dim = rng.choice(((64, 64), (128, 128), (128, 512), (64, 128), (256, 256), (128, 64)))
    if op == "append":
        batch, heads = rng.randint(1, 16), rng.choice((1, 2, 3, 8))
        tokens = _log(rng, 1, min(20000, 3 * 8160 * 640 // (batch * heads * (key_dim + value_dim))))
        return dict(op=op, dtype=dtype, batch=batch, heads=heads, key_dim=key_dim, value_dim=value_dim, tokens=tokens,
                    slots=tokens + rng.randint(0, 3 * tokens + 100), ragged=rng.random() < 0.6)
    heads = rng.choice((1, 2, 4, 8))
    batch = rng.randint(1, 6)
    if op == "evict":
        slots = _log(rng, 64, min(100000, 4 * 8 * 32768 * 200 // (batch * heads * (key_dim + value_dim))))
        keep = rng.randint(slots // 3 + 1, slots)
        return dict(op=op, dtype="bf16", batch=batch, heads=heads, key_dim=key_dim, value_dim=value_dim, slots=slots, keep=keep,
                    first=rng.randint(0, keep // 4), recent=rng.randint(0, keep // 2), ragged=rng.random() < 0.5)
    group = rng.choice((1, 2, 4, 5, 8))
    most_bank = min(150000, 4 * 8 * 131072 * 256 // (2 * batch * heads * (key_dim + value_dim)))
    if rng.random() < 0.5:
        tokens = rng.choice((1, 1, 2, 3, 5))
        slots = _log(rng, 16, most_bank)
    else:
        slots = _log(rng, 16, min(most_bank, 40000))
        most = 3 * 16 * 900 * 16384 * 256 // (batch * heads * group * slots * (key_dim + value_dim))
        tokens = _log(rng, 1, max(1, min(most, 2000, slots // 2)))
    return dict(op=op, dtype=dtype, batch=batch, q_heads=heads * group, heads=heads, key_dim=key_dim, value_dim=value_dim, tokens=tokens, slots=slots,
                fill=rng.randint((slots + 1) // 2, slots), ragged=rng.random() < 0.6, causal=rng.random() < 0.5, weigh=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ the lengths that go with a case
def _sections(case):
    return tuple(int(s) for s in case["axes"].split(","))


def _lens(case):
    """Filled slots of each stream: all alike, or falling to two thirds of the first one's."""
    fill = case.get("fill", case["slots"])
    return [max(1, fill - (b * fill // (3 * case["batch"]) if case["ragged"] else 0)) for b in range(case["batch"])]


def _counts(case):
    """Valid tokens of each stream in a padded batch."""
    return [max(1, case["tokens"] - (b * case["tokens"] // (2 * case["batch"]) if case["ragged"] else 0)) for b in range(case["batch"])]


def _row_bytes(case):
    return (case["key_dim"] + case["value_dim"]) * 17 // 32      # codes and block scales of one slot


def work(case):
    op = case["op"]
    if op in ("rotary", "norm_rotary"):
        rows = case["batch"] * case["tokens"] * (case["q_heads"] + case["k_heads"])
        passes = 3 if op == "norm_rotary" and case["grad"] else 2
        flops = (6 if op == "rotary" else 20 if case["grad"] else 10) * rows * case["dim"] // 2
        return {"bytes": passes * rows * case["dim"] * SIZE[case["dtype"]] + 12 * case["batch"] * case["tokens"], "flops": flops}
    dims = case["key_dim"] + case["value_dim"]
    if op == "append":
        rows = sum(_counts(case)) * case["heads"]
        return {"bytes": rows * (dims * SIZE[case["dtype"]] + 2 * _row_bytes(case) + 2 * dims), "flops": 4 * rows * dims}
    if op == "evict":
        kept = sum(min(case["keep"], n) for n in _lens(case)) * case["heads"]
        return {"bytes": 4 * sum(_lens(case)) * case["heads"] + kept * (3 * _row_bytes(case) + 2 * dims + 8), "flops": kept * dims}
    group = case["q_heads"] // case["heads"]
    pairs = 0
    for n, c in zip(_lens(case), _counts(case)):
        pairs += (c * n - c * (c - 1) // 2 if case["causal"] else c * n) * case["q_heads"]
    nbytes = sum(_lens(case)) * case["heads"] * (_row_bytes(case) + (8 if case["weigh"] else 0))
    nbytes += case["batch"] * case["tokens"] * case["heads"] * group * dims * SIZE[case["dtype"]]
    return {"bytes": nbytes, "flops": 2 * pairs * dims}


# ------------------------------------------------------------------------------------------------ inputs
def _randn(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _frequencies(case):
    """Radians a position for every channel pair (fp64), and the axis each pair turns with."""
    sections = _sections(case)
    total = sum(sections)
    freq, axis = [], []
    for a, n in enumerate(sections):
        for j in range(n):
            step = (len(freq), total) if case["shared"] else (j, n)
            freq.append(case["base"] ** (-step[0] / step[1]))
            axis.append(a)
    return torch.tensor(freq, dtype=torch.float64, device=DEVICE), torch.tensor(axis, device=DEVICE)


def _bank(case, gen, slots, lens):
    """A bank as a program holds it: `lens` slots filled, the rest memory that was never written."""
    b, h = case["batch"], case["heads"]
    bank = {"weight": torch.zeros((b, h, slots), device=DEVICE), "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE)}
    live = (torch.arange(slots, device=DEVICE) < bank["lens"][:, None]).view(b, 1, slots, 1)
    for name, dim in (("key", case["key_dim"]), ("value", case["value_dim"])):
        channel = torch.exp(0.5 * _randn(gen, (1, h, 1, dim)))       # channels of different spread, as trained projections have
        codes, scales = _quantize(_randn(gen, (b, h, slots, dim)) * channel)
        dirt = torch.randint(0, 256, (slots, 1), generator=gen, device=DEVICE).to(torch.uint8)
        bank[name + "_codes"] = torch.where(live, codes, dirt)
        bank[name + "_scales"] = torch.where(live, scales, dirt)
    return bank


def _handle(bank):
    from mivos_amd import ops
    return ops.Bank4(bank["key_codes"], bank["key_scales"], bank["value_codes"], bank["value_scales"], bank["weight"], bank["lens"])


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    op, state = case["op"], dict(case=case)
    if op in ("rotary", "norm_rotary"):
        b, n, hq, hk, d = (case[k] for k in ("batch", "tokens", "q_heads", "k_heads", "dim"))
        dtype = TYPES[case["dtype"]]
        joint = _randn(gen, (b, n, (hq + 2 * hk) * d), dtype)        # one projection's output: q | k | v
        state["q"] = joint[..., :hq * d].view(b, n, hq, d)
        state["k"] = joint[..., hq * d:(hq + hk) * d].view(b, n, hk, d)
        i = torch.arange(n, device=DEVICE)
        start = torch.randint(0, 64, (b, 1), generator=gen, device=DEVICE) + case["time0"]
        w, h = case["width"], case["height"]
        state["positions"] = torch.stack([start + i // (w * h), ((i // w) % h).expand(b, n), (i % w).expand(b, n)], -1).to(torch.int32).contiguous()
        state["freq"], state["axis"] = _frequencies(case)
        if op == "norm_rotary":
            state["q_weight"], state["k_weight"] = 1 + 0.3 * _randn(gen, (d,)), 1 + 0.3 * _randn(gen, (d,))
        if case["grad"]:
            state["dq"], state["dk"] = _randn(gen, (b, n, hq, d), dtype), _randn(gen, (b, n, hk, d), dtype)
        if own:
            from mivos_amd import ops
            state["plan"] = ops.RotaryAxes(d, _sections(case), base=case["base"], shared=case["shared"], interleaved=case["interleaved"], device=DEVICE)
        return state
    b, h = case["batch"], case["heads"]
    if op == "append":
        counts = _counts(case)
        room = [case["slots"] - case["tokens"] - (i * (case["slots"] - case["tokens"]) // (2 * b) if case["ragged"] else 0) for i in range(b)]
        state["bank"] = _bank(case, gen, case["slots"], room)
        state["at"] = torch.tensor(room, dtype=torch.int32, device=DEVICE)
        state["count"] = torch.tensor(counts, dtype=torch.int32, device=DEVICE)
        dtype = TYPES[case["dtype"]]
        state["keys"] = _randn(gen, (b, case["tokens"], h, case["key_dim"]), dtype)
        state["values"] = _randn(gen, (b, case["tokens"], h, case["value_dim"]), dtype)
    elif op == "read":
        state["bank"] = _bank(case, gen, case["slots"], _lens(case))
        # as an earlier pass of as many queries has left it
        earlier = torch.rand((b, h, case["slots"]), generator=gen, device=DEVICE)
        state["bank"]["weight"] = earlier * (2.0 * case["tokens"] * case["q_heads"] / h / case["fill"])
        state["queries"] = (1.5 * _randn(gen, (b, case["tokens"], case["q_heads"], case["key_dim"]))).to(TYPES[case["dtype"]])
        state["count"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEVICE)
    else:
        state["bank"] = _bank(case, gen, case["slots"], _lens(case))
        weight = torch.exp(2 * _randn(gen, (b, h, case["slots"])) - 4)
        # what no query has looked at yet has received nothing: many equal weights
        state["bank"]["weight"] = torch.where(torch.rand((b, h, case["slots"]), generator=gen, device=DEVICE) < 0.1, torch.zeros_like(weight), weight)
        state["out"] = _bank(case, gen, case["keep"], [1] * b)
        if own:
            state["out_handle"] = _handle(state["out"])
    if own:
        state["handle"] = _handle(state["bank"])
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _quantize(x):
    """fp32 [..., D] -> (codes [..., D/2], scales [..., D/32]) as uint8."""
    blocks = x.float().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    mantissa, exponent = torch.frexp(torch.where(bad, torch.zeros_like(top), top))
    e = torch.where(top > 0, exponent - 3 + (mantissa > 0.75).int(), torch.full_like(exponent, -120)).clamp(-120, 125)
    a = torch.ldexp(blocks, -e)
    m = a.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)).to(torch.uint8)
    code = torch.where(bad, torch.zeros_like(code), code | (torch.signbit(a).to(torch.uint8) << 3)).flatten(-2)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale[..., 0].to(torch.uint8)


def _unpack(codes, scales):
    """The values that codes and scales stand for, fp32."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    e = scales.int()
    scale = torch.where(e == 255, torch.full_like(e, 0, dtype=torch.float32) + math.nan, torch.ldexp(torch.ones_like(e, dtype=torch.float32), e - 127))
    return (level[c.int()].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _angles(state):
    return (state["positions"].double()[..., state["axis"]] * state["freq"])[..., None, :]      # [B, N, 1, pairs]


def _turn(x, angle, interleaved):
    """Rotates channel pairs by `angle`; channels beyond the pairs pass."""
    p = angle.shape[-1]
    cos, sin = torch.cos(angle).to(x.dtype), torch.sin(angle).to(x.dtype)
    head, rest = x[..., :2 * p], x[..., 2 * p:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :p], head[..., p:])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1), rest], -1)


def _norm(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _norm_grad(g, x, weight):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    gw = g * weight
    dx = r * (gw - x * (r * r) * (gw * x).mean(-1, keepdim=True))
    return dx, (g * x * r).sum((0, 1, 2))


def _plain_rotary(state):
    case, angle = state["case"], _angles(state)
    turn = lambda x, s: _turn(x.float(), s * angle, case["interleaved"])  # noqa: E731
    if case["op"] == "rotary":
        names = ("dq", "dk") if case["grad"] else ("q", "k")
        return tuple(turn(state[n], -1.0 if case["grad"] else 1.0).to(state[n].dtype) for n in names)
    if not case["grad"]:
        return tuple(turn(_norm(state[n].float(), state[n + "_weight"]), 1.0).to(state[n].dtype) for n in ("q", "k"))
    (dq, dwq), (dk, dwk) = (_norm_grad(turn(state["d" + n], -1.0), state[n].float(), state[n + "_weight"]) for n in ("q", "k"))
    return dq.to(state["q"].dtype), dk.to(state["k"].dtype), dwq, dwk


def _plain_values(bank, first, count, lens):
    """bf16 values of slots [first, first + count) of every stream; zeros behind its length."""
    slots = first.long()[:, None] + torch.arange(count, device=first.device)                     # [B, count]
    live = (slots < lens.long()[:, None])[:, None, :, None]
    outs = []
    for name in ("key", "value"):
        pick = slots.clamp(max=bank[name + "_codes"].shape[2] - 1)[:, None, :, None]
        rows = [torch.take_along_dim(bank[name + kind], pick, 2) for kind in ("_codes", "_scales")]
        values = _unpack(*rows)
        outs.append(torch.where(live, values, torch.zeros_like(values)).to(torch.bfloat16))
    return outs


def _plain_append(state):
    bank, at, count = state["bank"], state["at"].long(), state["count"].long()
    b, n = state["keys"].shape[:2]
    slots = at[:, None] + torch.arange(n, device=at.device)
    valid = (torch.arange(n, device=at.device) < count[:, None])[:, :, None, None]
    row = torch.arange(b, device=at.device)[:, None]
    for name, x in (("key", state["keys"]), ("value", state["values"])):
        for kind, new in zip(("_codes", "_scales"), _quantize(x)):
            old = bank[name + kind]
            old[row, :, slots] = torch.where(valid, new, old[row, :, slots])
    old = bank["weight"]
    old[row, :, slots] = torch.where(valid[..., 0], torch.zeros_like(old[row, :, slots]), old[row, :, slots])
    lens = bank["lens"].copy_(at + count)
    return (*_plain_values(bank, state["at"], n, lens), lens)


def _plain_read(state):
    case, bank, q = state["case"], state["bank"], state["queries"]
    b, n, hq, d = q.shape
    h, s = case["heads"], case["slots"]
    g = hq // h
    lens, count = bank["lens"].long().view(b, 1, 1), state["count"].long().view(b, 1, 1)
    slot, token = torch.arange(s, device=q.device), torch.arange(n, device=q.device).view(1, n, 1)
    last = (lens - count + token).clamp(max=s) if case["causal"] else lens - 1
    seen = (slot <= last) & (slot < lens) & (token < count)                                      # [B, N, S]
    seen = seen[:, None, :, None, :].expand(b, 1, n, g, s).reshape(b, 1, n * g, s)
    rows = q.float().view(b, n, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, n * g, d)
    live = (slot < lens)[..., None]                                                              # [B, 1, S, 1]
    keys, values = (_unpack(bank[k + "_codes"], bank[k + "_scales"]) for k in ("key", "value"))
    keys, values = torch.where(live, keys, torch.zeros_like(keys)), torch.where(live, values, torch.zeros_like(values))
    logits = torch.matmul(rows, keys.transpose(2, 3)) * d ** -0.5
    logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p, values).view(b, h, n, g, -1).permute(0, 2, 1, 3, 4).reshape(b, n, hq, -1).to(q.dtype)
    if not case["weigh"]:
        return out
    return out, bank["weight"].add_(p.sum(2))


def _plain_evict(state):
    case, bank, out = state["case"], state["bank"], state["out"]
    keep, s = case["keep"], case["slots"]
    lens = bank["lens"].long().view(-1, 1, 1)
    slot = torch.arange(s, device=lens.device)
    weight = bank["weight"]
    safe = (slot < lens) & ((slot < case["first"]) | (slot >= lens - case["recent"]))
    rank = torch.where(safe, torch.full_like(weight, math.inf), torch.where(slot < lens, weight, torch.full_like(weight, -1.0)))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]           # equal weights: the lowest slot stays
    fresh = torch.minimum(lens, torch.full_like(lens, keep))
    valid = torch.arange(keep, device=lens.device) < fresh                                       # [B, 1, keep]
    slots = torch.sort(torch.where(valid, order, torch.full_like(order, s)), dim=-1).values
    pick = slots.clamp(max=s - 1)
    for name in ("key_codes", "key_scales", "value_codes", "value_scales"):
        out[name].copy_(torch.where(valid[..., None], torch.take_along_dim(bank[name], pick[..., None], 2), out[name]))
    out["weight"].copy_(torch.where(valid, torch.take_along_dim(weight, pick, 2), out["weight"]))
    out["lens"].copy_(fresh.view(-1))
    slots = torch.where(valid, slots, torch.full_like(slots, -1)).to(torch.int32)
    return (slots, out["lens"], out["weight"], *_plain_values(out, torch.zeros_like(out["lens"]), keep, out["lens"]))


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(state):
    from mivos_amd import ops
    case = state["case"]
    op = case["op"]
    if op == "rotary":
        if case["grad"]:
            return ops.rotary_axes_grad(state["dq"], state["dk"], state["positions"], state["plan"])
        return ops.rotary_axes(state["q"], state["k"], state["positions"], state["plan"])
    if op == "norm_rotary":
        weights = state["q_weight"], state["k_weight"], state["positions"], state["plan"]
        if case["grad"]:
            return ops.norm_rotary_grad(state["dq"], state["dk"], state["q"], state["k"], *weights, eps=EPS)
        return ops.norm_rotary(state["q"], state["k"], *weights, eps=EPS)
    bank = state["handle"]
    if op == "append":
        ops.bank4_append(bank, state["keys"], state["values"], at=state["at"], count=state["count"])
        return (*ops.bank4_values(bank, first=state["at"], count=case["tokens"]), bank.lens)
    if op == "read":
        out = ops.bank4_read(bank, state["queries"], causal=case["causal"], count=state["count"], weigh=case["weigh"])
        return (out, bank.weight) if case["weigh"] else out
    out = state["out_handle"]
    slots = ops.bank4_evict(bank, case["keep"], out, first=case["first"], recent=case["recent"])
    return (slots, out.lens, out.weight, *ops.bank4_values(out, count=case["keep"]))


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"rotary": _plain_rotary, "norm_rotary": _plain_rotary, "append": _plain_append, "read": _plain_read, "evict": _plain_evict}[op](state)


# ------------------------------------------------------------------------------------------------ 64 bits, by the definitions
def _exact_grid(x):
    """The values a 4-bit row stands for: the nearest point of each block's grid, in fp64."""
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[-1], 32):
        block = x[..., c:c + 32]
        top = block.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top / 6)).clamp(-120, 125)         # then put right where log2 lies next to a whole number
        e = torch.where(6 * torch.exp2(e - 1) >= top, e - 1, e)
        e = torch.where(6 * torch.exp2(e) < top, e + 1, e).clamp(-120, 125)
        unit = torch.exp2(e)
        a = block / unit
        step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
        out[..., c:c + 32] = (torch.round(a / step) * step).clamp(-6, 6) * unit
    return out


def _exact_unpack(codes, scales):
    low, high = (codes & 15).double(), (codes >> 4).double()
    c = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device=codes.device)
    c[..., 0::2], c[..., 1::2] = low, high
    sign = 1 - 2 * (c >= 8).double()
    c = c % 8
    e, m = torch.floor(c / 2), c % 2
    value = torch.where(e == 0, 0.5 * m, torch.exp2(e - 1) * (1 + 0.5 * m))
    return sign * value * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _exact_rotary(state):
    case = state["case"]
    sections, total = _sections(case), sum(_sections(case))
    q, k = (state["dq"], state["dk"]) if case["grad"] else (state["q"], state["k"])
    sign = -1.0 if case["grad"] else 1.0
    outs, extra = [], []
    for x, name in ((q, "q"), (k, "k")):
        x = x.double()
        if case["op"] == "norm_rotary" and not case["grad"]:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * state[name + "_weight"].double()
        y = x.clone()
        i = 0
        for a, n in enumerate(sections):
            for j in range(n):
                exponent = i / total if case["shared"] else j / n
                t = sign * state["positions"][..., a, None].double() / case["base"] ** exponent
                u, v = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + total)
                z = torch.complex(x[..., u], x[..., v]) * torch.polar(torch.ones_like(t), t)
                y[..., u], y[..., v] = z.real, z.imag
                i += 1
        if case["op"] == "norm_rotary" and case["grad"]:
            z, w = state[name].double(), state[name + "_weight"].double()
            rms = torch.sqrt(z.square().mean(-1, keepdim=True) + EPS)
            unit = z / rms
            extra.append((y * unit).sum((0, 1, 2)))
            y = y * w
            y = (y - unit * (y * unit).mean(-1, keepdim=True)) / rms
        outs.append(y)
    return (*outs, *extra)


def _exact_read(state):
    case, bank, q = state["case"], state["bank"], state["queries"].double()
    b, n, hq, d = q.shape
    g = hq // case["heads"]
    out = torch.zeros((b, n, hq, case["value_dim"]), dtype=torch.float64, device=q.device)
    weight = bank["weight"].double()
    for i, (size, count) in enumerate(zip(_lens(case), _counts(case))):
        for h in range(case["heads"]):
            keys, values = (_exact_unpack(bank[k + "_codes"][i, h, :size], bank[k + "_scales"][i, h, :size]) for k in ("key", "value"))
            for j in range(h * g, h * g + g):
                a = q[i, :count, j] @ keys.t() / math.sqrt(d)
                if case["causal"]:
                    hidden = torch.arange(size, device=q.device)[None] > (size - count + torch.arange(count, device=q.device))[:, None]
                    a = a.masked_fill(hidden, -math.inf)
                a = torch.exp(a - torch.clamp(a.amax(-1, keepdim=True), min=-1e300))
                total = a.sum(-1, keepdim=True)
                a = a / torch.where(total > 0, total, 1.0)
                out[i, :count, j] = a @ values
                weight[i, h, :size] += a.sum(0)
    return (out, weight) if case["weigh"] else out


def _exact_evict(state):
    case, bank, out = state["case"], state["bank"], state["out"]
    keep, dims = case["keep"], (case["key_dim"], case["value_dim"])
    shape = out["weight"].shape
    weight = out["weight"].double().clone()
    values = [torch.zeros((*shape, d), dtype=torch.float64, device=weight.device) for d in dims]
    for i, size in enumerate(_lens(case)):
        for h in range(case["heads"]):
            w = bank["weight"][i, h, :size].double()
            slot = torch.arange(size, device=w.device)
            w = torch.where((slot < case["first"]) | (slot >= size - case["recent"]), math.inf, w)
            stays = slot
            if size > keep:
                line = torch.topk(w, keep).values[-1]                # the keep-th largest weight
                above, level = slot[w > line], slot[w == line]
                stays = torch.cat([above, level[:keep - above.numel()]]).sort().values
            weight[i, h, :stays.numel()] = bank["weight"][i, h, stays].double()
            for v, k in zip(values, ("key", "value")):
                v[i, h, :stays.numel()] = _exact_unpack(bank[k + "_codes"][i, h, stays], bank[k + "_scales"][i, h, stays])
    return (None, None, weight, *values)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("rotary", "norm_rotary"):
        return _exact_rotary(state)
    if op == "read":
        return _exact_read(state)
    if op == "evict":
        return _exact_evict(state)
    outs = []
    valid = (torch.arange(case["tokens"], device=DEVICE) < state["count"].long()[:, None])[:, None, :, None]
    for x in (state["keys"], state["values"]):
        outs.append(torch.where(valid, _exact_grid(x).transpose(1, 2), 0.0))
    return (*outs, None)
