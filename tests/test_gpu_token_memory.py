"""Token-memory operators on an MI355X against the fp64 oracle (oracle/token_memory.py).

Tolerances, element by element (u = 2^-24, h = half a step of the type: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32; denormal fp16 outputs add half
of 2^-24):
  rotation   h |y| + 2^-19 a, a = the pair's length: sine / cosine 4u, products and sum 3u, mean of at most 512 squares 12u, root and scale 5u
             = 24u < 2^-19.
  4-bit rows equality: every step up to the rounding is exact, and so is the rounding.
  read       (h + P) |out| + (P + 2 d + 2^-20) sum p |v|, P = the rounding of the weights p (2^-8, 2^-16, 2^-24 for bf16, fp16, fp32 queries),
             d = (Dk parts + 16) u A, the error of a logit with A = max sum |q| |k| scale (x log2 e folded: the factor 2).
  weight     (2 d + 2^-20 + rows u) of the value, and 2^-126 a row: the exponential gives 0 below the smallest normal fp32 number, so each
             row's share is off by less than that number (1.18e-38); for the same reason a read's elements by slots 2^-126 max |v|, below 6 * 2^8 here."""
import math

import pytest
import torch

from mivos_amd import ops
from mivos_amd._lib import MivosHipError
from oracle import token_memory as O

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
PART = {torch.bfloat16: (2.0 ** -8, 1), torch.float16: (2.0 ** -16, 2), torch.float32: (2.0 ** -24, 3)}
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _within(got, ref, tol):
    most, got = torch.finfo(got.dtype).max, got.double().cpu()
    assert got.shape == ref.shape
    assert torch.equal(got.isnan(), ref.isnan())
    ok = ref.isnan() | ((got - ref).abs() <= tol + 1e-300) | (got.isinf() & (got.sign() == ref.sign()) & (ref.abs() + tol >= most))      # (beyond the type: infinity)
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off, worst ratio {float(((got - ref).abs() / (tol + 1e-300)).nan_to_num(0).max()):.3g}"


# ------------------------------------------------------------------------------------------------ rotary
# dim, sections, interleaved, shared, batch, tokens, q heads, k heads
ROTARY = [
    (128, (16, 24, 24), False, False, 2, 37, 4, 2),
    (64, (8, 12, 12), True, False, 8, 1, 8, 2),
    (80, (8, 16, 16), False, False, 3, 41, 5, 5),
    (96, (16, 8, 8), True, True, 1, 130, 3, 1),           # 32 channels behind the pairs
    (128, (40,), False, False, 1, 5, 2, 2),               # one axis, 48 channels behind
    (72, (9, 13, 14), False, True, 2, 19, 3, 3),          # no multiple of 16
    (34, (3, 2), True, False, 1, 7, 1, 1),
    (2, (1,), False, False, 1, 3, 2, 1),
    (256, (0, 64, 64), False, False, 1, 33, 2, 0),        # an axis without pairs, no keys
    (512, (64, 96, 96), True, False, 1, 9, 2, 1),
    (130, (20, 20, 25), False, False, 1, 70, 2, 1),
    (16, (8,), False, False, 5, 611, 1, 1),               # more tokens than one tile
    (32, (2, 7, 7), True, False, 1, 17000, 2, 1),         # tiles of 16 tokens, the last one short
]


def _rotary_inputs(case, dtype, joint, seed=0):
    d, sections, inter, shared, b, n, hq, hk = case
    g = torch.Generator().manual_seed(seed + d + n)
    if joint:                                             # slices of one projection: token rows far apart
        x = torch.randn(b, n, (hq + 2 * hk) * d, generator=g).to(dtype)
        q, k = x[..., :hq * d].view(b, n, hq, d), x[..., hq * d:(hq + hk) * d].view(b, n, hk, d)
    else:
        q, k = torch.randn(b, n, hq, d, generator=g).to(dtype), torch.randn(b, n, hk, d, generator=g).to(dtype)
    pos = torch.randint(-40, 70000, (b, n, len(sections)), generator=g, dtype=torch.int32)
    pos[0, 0] = 2 ** 31 - 1
    pos[-1, -1] = -2 ** 31
    plan = ops.RotaryAxes(d, sections, base=1000.0, shared=shared, interleaved=inter, device=DEV)
    return g, q, (k if hk else None), pos, plan, O.angles(pos, sections, 1000.0, shared)


def _to_dev(t, joint):
    """Moves a tensor to the GPU keeping the strides of a slice of a joint projection."""
    if t is None or not joint:
        return None if t is None else t.to(DEV)
    base = torch.empty(t.untyped_storage().nbytes() // t.element_size(), dtype=t.dtype, device=DEV)
    base.copy_(torch.empty(0, dtype=t.dtype).set_(t.untyped_storage()))
    return base.as_strided(t.shape, t.stride(), t.storage_offset())


def _pair_length(y, pairs, inter):
    a = y.abs().clone()
    u = torch.arange(pairs) * 2 if inter else torch.arange(pairs)
    v = u + 1 if inter else u + pairs
    a[..., u] = a[..., v] = torch.sqrt(y[..., u].square() + y[..., v].square())
    return a


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: f"{c[0]}-{sum(c[1])}x{len(c[1])}-{c[5]}")
def test_rotary_axes_and_norm(case, dtype):
    d, sections, inter = case[:3]
    for joint in (False, True):
        g, q, k, pos, plan, angle = _rotary_inputs(case, dtype, joint)
        wq, wk = 1 + 0.3 * torch.randn(d, generator=g), 1 + 0.3 * torch.randn(d, generator=g)
        dq, dk, dpos = _to_dev(q, joint), _to_dev(k, joint), pos.to(DEV)
        for name, got, ref in (
                ("turn", ops.rotary_axes(dq, dk, dpos, plan), lambda x, w: O.turn(x, angle, inter)),
                ("back", ops.rotary_axes_grad(dq, dk, dpos, plan), lambda x, w: O.turn(x, -angle, inter)),
                ("norm", ops.norm_rotary(dq, dk, wq.to(DEV), None if k is None else wk.to(DEV), dpos, plan, eps=1e-5),
                 lambda x, w: O.norm_rotary(x, w.double(), angle, inter, 1e-5))):
            for y, x, w in zip(got, (q, k), (wq, wk)):
                if x is None:
                    assert y is None
                    continue
                assert y.dtype == dtype and y.is_contiguous()
                r = ref(x.double(), w)
                _within(y, r, HALF[dtype] * r.abs() + 2.0 ** -19 * _pair_length(r, plan.pairs, inter) + FLOOR[dtype])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: f"{c[0]}-{sum(c[1])}x{len(c[1])}-{c[5]}")
def test_norm_rotary_gradients(case, dtype):
    """dx: |dx| h + 2^-18 r (|w g| + |x| r^2 sum |w g x| / D) with the lengths of pairs for g; dw: sum |g x r| 2^-15 (a lane adds at most 128
    rows in turn here, then 256 / lanes shares and 16 + 64 workgroups: fewer than 512 = 2^9 roundings of u)."""
    d, sections, inter = case[:3]
    for joint in (False, True):
        g, q, k, pos, plan, angle = _rotary_inputs(case, dtype, joint, seed=5)
        ws = [1 + 0.3 * torch.randn(d, generator=g) for _ in range(2)]
        gs = [None if x is None else torch.randn(x.shape, generator=g).to(dtype) for x in (q, k)]
        dev = [_to_dev(x, joint) for x in (q, k)]
        got = ops.norm_rotary_grad(gs[0].to(DEV), None if k is None else gs[1].to(DEV), *dev, ws[0].to(DEV), None if k is None else ws[1].to(DEV),
                                   pos.to(DEV), plan, eps=1e-5)
        again = ops.norm_rotary_grad(gs[0].to(DEV), None if k is None else gs[1].to(DEV), *dev, ws[0].to(DEV), None if k is None else ws[1].to(DEV),
                                     pos.to(DEV), plan, eps=1e-5)
        for a, b in zip(got, again):
            assert a is b is None or torch.equal(a, b)              # a fixed order of additions
        for i, x in enumerate((q, k)):
            if x is None:
                assert got[i] is None and got[2 + i] is None
                continue
            x, w, dy = x.double(), ws[i].double(), gs[i].double()
            dx, dw = O.norm_rotary_grad(dy, x, w, angle, inter, 1e-5)
            r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
            ga = _pair_length(O.turn(dy, -angle, inter), plan.pairs, inter)
            _within(got[i], dx, HALF[dtype] * dx.abs() + 2.0 ** -18 * r * (ga * w.abs() + x.abs() * r * r * (ga * w.abs() * x.abs()).mean(-1, keepdim=True)) + FLOOR[dtype])
            _within(got[2 + i], dw, 2.0 ** -15 * (ga * x.abs() * r).sum((0, 1, 2)))


def test_norm_rotary_gradient_against_differences():
    """The kernels' gradient of sum(y c) along random directions against central differences of the oracle's forward pass in fp64 (their own
    error: h^2 = 1e-10 of the third derivative; the gradient's: 2^-18 of the terms, fp32)."""
    case = (64, (8, 12, 12), False, False, 2, 9, 3, 2)
    g, q, k, pos, plan, angle = _rotary_inputs(case, torch.float32, False)
    w = 1 + 0.3 * torch.randn(64, generator=g)
    c = torch.randn(q.shape, generator=g)
    dx, _, dw, _ = ops.norm_rotary_grad(c.to(DEV), None, q.to(DEV), None, w.to(DEV), None, pos.to(DEV), plan, eps=1e-3)
    f = lambda x, w: (O.norm_rotary(x, w, angle, False, 1e-3) * c.double()).sum()  # noqa: E731
    for _ in range(4):
        u, v = torch.randn(q.shape, generator=g, dtype=torch.float64), torch.randn(64, generator=g, dtype=torch.float64)
        slope = (f(q.double() + 1e-5 * u, w.double() + 1e-5 * v) - f(q.double() - 1e-5 * u, w.double() - 1e-5 * v)) / 2e-5
        got = (dx.double().cpu() * u).sum() + (dw.double().cpu() * v).sum()
        size = (dx.double().cpu() * u).abs().sum() + (dw.double().cpu() * v).abs().sum()
        assert abs(got - slope) <= 2.0 ** -16 * size


def test_rotary_empty_and_broadcast_positions():
    plan = ops.RotaryAxes(64, (8, 12, 12), device=DEV)
    q = torch.randn(0, 5, 2, 64, device=DEV)
    y, _ = ops.rotary_axes(q, None, torch.zeros(0, 5, 3, dtype=torch.int32, device=DEV), plan)
    assert y.shape == q.shape
    w = torch.ones(64, device=DEV)
    gq, gk, gw, _ = ops.norm_rotary_grad(q, None, q, None, w, None, torch.zeros(0, 5, 3, dtype=torch.int32, device=DEV), plan)
    assert gq.shape == q.shape and float(gw.abs().max()) == 0
    q = torch.randn(3, 50, 2, 64, device=DEV)
    one = torch.randint(0, 99, (1, 50, 3), dtype=torch.int32, device=DEV)
    a = ops.rotary_axes(q, None, one.expand(3, 50, 3), plan)[0]
    assert torch.equal(a, ops.rotary_axes(q, None, one.repeat(3, 1, 1), plan)[0])
    b = ops.rotary_axes(q, None, one.repeat(3, 1, 1).transpose(1, 2).contiguous().transpose(1, 2), plan)[0]
    assert torch.equal(a, b)
    off = torch.randn(3 * 50 * 2 * 64 + 1, device=DEV)[1:].view(3, 50, 2, 64)       # not 16-byte aligned: the other kernel
    ref = ops.rotary_axes(off.clone(), None, one.expand(3, 50, 3), plan)[0]
    assert float((ops.rotary_axes(off, None, one.expand(3, 50, 3), plan)[0] - ref).abs().max()) <= 2.0 ** -19 * float(off.abs().max()) * 2


def test_norm_rotary_gradient_without_key_heads():
    """Keys of no heads: their weight's gradient is a sum over nothing, 0, whatever its memory held; both kernels."""
    for dim in (64, 40):
        plan, w = ops.RotaryAxes(dim, (8,), device=DEV), torch.ones(dim, device=DEV)
        q, pos = torch.randn(2, 5, 2, dim, device=DEV), torch.zeros(2, 5, 1, dtype=torch.int32, device=DEV)
        k = q[:, :, :0]
        for t in [torch.full((dim,), float("nan"), device=DEV) for _ in range(8)]:      # (what the allocator hands out next)
            del t
        _, gk, gw, kw = ops.norm_rotary_grad(q, k, q, k, w, w, pos, plan)
        assert gk.shape == k.shape and torch.equal(kw, torch.zeros_like(w))
        assert torch.equal(gw, ops.norm_rotary_grad(q, None, q, None, w, None, pos, plan)[2])


def test_norm_rotary_zero_rows():
    """A row of zeros: eps alone holds the norm; its gradient is w g / sqrt(eps)."""
    plan = ops.RotaryAxes(64, (32,), device=DEV)
    z, w = torch.zeros(1, 2, 1, 64, device=DEV), torch.ones(64, device=DEV)
    pos = torch.zeros(1, 2, 1, dtype=torch.int32, device=DEV)
    assert float(ops.norm_rotary(z, None, w, None, pos, plan, eps=1e-6)[0].abs().max()) == 0
    dx = ops.norm_rotary_grad(torch.ones_like(z), None, z, None, w, None, pos, plan, eps=1e-6)[0]
    assert float((dx * 1e-3 - 1).abs().max()) < 1e-5


# ------------------------------------------------------------------------------------------------ the bank
def _dirty(batch, heads, slots, dk, dv, seed=0):
    """A bank whose memory was never written: random bytes, NaN scales among them."""
    bank = ops.Bank4.empty(batch, heads, slots, dk, dv, device=DEV)
    g = torch.Generator().manual_seed(seed)
    for t in (bank.key_codes, bank.key_scales, bank.value_codes, bank.value_scales):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    bank.key_scales[..., ::3, :] = 255
    bank.value_scales[..., ::3, :] = 255
    return bank


def _rows(bank):
    """fp64 rows as the bank's bytes stand for them."""
    return (O.unpack(bank.key_codes.cpu(), bank.key_scales.cpu()), O.unpack(bank.value_codes.cpu(), bank.value_scales.cpu()))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dk,dv,heads,tokens", [(64, 64, 3, 1), (128, 512, 1, 33), (32, 96, 2, 300), (1024, 32, 1, 7)])
def test_append_and_values(dtype, dk, dv, heads, tokens):
    g = torch.Generator().manual_seed(dk + tokens)
    bank = _dirty(3, heads, 2 * tokens + 5, dk, dv)
    before = [t.clone() for t in (bank.key_codes, bank.key_scales, bank.value_codes, bank.value_scales)]
    bank.weight.fill_(3.0)
    x = [torch.randn(3, tokens, heads, d, generator=g) * torch.exp(4 * torch.randn(3, tokens, heads, d // 32, 1, generator=g)).expand(-1, -1, -1, -1, 32).flatten(-2)
         for d in (dk, dv)]
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])          # ties
    x[0][0, 0, 0, :32] = torch.cat([grid, -grid, 2 * grid, 6 - grid])
    x[0][1, 0, 0, :32] = 0
    x[0][1, tokens - 1, 0, 0] = -0.0
    x[1][2, 0, 0, 5] = float("inf")
    x[1][1, 0, 0, 3] = float("nan")
    x = [t.to(dtype) for t in x]
    at = torch.tensor([0, 5, tokens + 5], dtype=torch.int32)
    count = torch.tensor([tokens, tokens, max(1, tokens // 2)], dtype=torch.int32)
    ops.bank4_append(bank, x[0].to(DEV), x[1].to(DEV), at=at.to(DEV), count=count.to(DEV))
    assert bank.lens.tolist() == (at + count).tolist()
    touched = torch.zeros(3, heads, bank.slots, dtype=torch.bool)
    for b in range(3):
        touched[b, :, int(at[b]):int(at[b] + count[b])] = True
    for d, rows, codes, scales, old in ((dk, x[0], bank.key_codes, bank.key_scales, before[:2]), (dv, x[1], bank.value_codes, bank.value_scales, before[2:])):
        c, s = O.quantise(rows.double())
        for b in range(3):
            sl = slice(int(at[b]), int(at[b] + count[b]))
            assert torch.equal(codes[b, :, sl].cpu(), O.pack(c[b, :int(count[b])]).transpose(0, 1))
            assert torch.equal(scales[b, :, sl].cpu(), s[b, :int(count[b])].transpose(0, 1).to(torch.uint8))
        assert torch.equal(codes.cpu()[~touched], old[0].cpu()[~touched]) and torch.equal(scales.cpu()[~touched], old[1].cpu()[~touched])
    assert torch.equal(bank.weight.cpu() == 0, touched) and int(bank.status.abs().sum()) == 0
    for out_dtype in (torch.float32, torch.bfloat16):
        for first, n in ((None, bank.slots), (at.to(DEV) - 2, tokens + 1)):
            got = ops.bank4_values(bank, first=first, count=n, dtype=out_dtype)
            for y, ref in zip(got, _rows(bank)):
                full = torch.zeros(3, heads, n, ref.shape[3], dtype=torch.float64)
                for b in range(3):
                    for j in range(n):
                        slot = j + (0 if first is None else int(first[b]))
                        if 0 <= slot < int(bank.lens[b]):
                            full[b, :, j] = ref[b, :, slot]
                full = full.to(out_dtype).double()           # never-written bytes can say 6 * 2^127: beyond either type, infinity
                assert y.dtype == out_dtype and torch.equal(y.double().cpu().nan_to_num(7e77), full.nan_to_num(7e77))


def test_append_strides_behind_each_other_and_overflow():
    """Slices of a joint projection, an unaligned operand, `at` = the bank's own lengths, and tokens that do not fit."""
    bank, plain = ops.Bank4.empty(2, 2, 20, 64, 32, device=DEV), ops.Bank4.empty(2, 2, 20, 64, 32, device=DEV)
    g = torch.Generator().manual_seed(1)
    joint = torch.randn(2, 7, 2 * 96 + 3, generator=g).to(DEV)
    k, v = joint[..., :128].view(2, 7, 2, 64), joint[..., 129:193].view(2, 7, 2, 32)
    for step in range(2):
        ops.bank4_append(bank, k, v, count=torch.tensor([7, 4], dtype=torch.int32, device=DEV))
        ops.bank4_append(plain, k.contiguous(), v.contiguous(), at=torch.tensor([7 * step, 4 * step], dtype=torch.int32, device=DEV),
                         count=torch.tensor([7, 4], dtype=torch.int32, device=DEV))
    assert bank.lens.tolist() == plain.lens.tolist() == [14, 8]
    for a, b in zip(ops.bank4_values(bank, dtype=torch.float32), ops.bank4_values(plain, dtype=torch.float32)):
        assert torch.equal(a, b) and float(a[0, :, :14].abs().amin(-1).max()) >= 0
    bank.check_room()
    ops.bank4_append(bank, k, v)                                  # 14 + 7 > 20
    assert bank.lens.tolist() == [20, 15]
    with pytest.raises(MivosHipError, match="did not fit"):
        bank.check_room()
    bank.check_room()
    ops.bank4_append(bank, k, v, at=torch.tensor([-3, 100], dtype=torch.int32, device=DEV))
    assert bank.lens.tolist() == [4, 20]
    with pytest.raises(MivosHipError, match="did not fit"):
        bank.check_room()
    ops.bank4_append(bank, k[:, :0], v[:, :0])
    assert bank.lens.tolist() == [4, 20]


def _filled(batch, heads, slots, dk, dv, lens, seed=0, spread=1.0):
    """A dirty bank with `lens` slots filled from normal rows."""
    bank = _dirty(batch, heads, slots, dk, dv, seed)
    g = torch.Generator().manual_seed(seed + 1)
    n = max(lens)
    if n:
        ops.bank4_append(bank, (spread * torch.randn(batch, n, heads, dk, generator=g)).to(DEV), torch.randn(batch, n, heads, dv, generator=g).to(DEV),
                         at=torch.zeros(batch, dtype=torch.int32, device=DEV), count=torch.tensor(lens, dtype=torch.int32, device=DEV))
    for b in range(batch):                                        # what lies behind a stream's length is nobody's
        bank.key_scales[b, :, lens[b]:] = 255
        bank.value_scales[b, :, lens[b]:] = 255
    bank.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    return bank


def _check_read(bank, q, causal, count, weigh, scale=None, dev_q=None):
    keys, values = _rows(bank)
    b, t, hq, d = q.shape
    cnt = torch.full((b,), t) if count is None else count
    s = d ** -0.5 if scale is None else scale
    ref, received, mag, big = O.read(keys, values, bank.lens.cpu(), q.double(), cnt, s, causal)
    base = bank.weight.double().cpu()
    got = ops.bank4_read(bank, q.to(DEV) if dev_q is None else dev_q, scale=scale, causal=causal, count=None if count is None else count.to(DEV), weigh=weigh)
    assert got.dtype == q.dtype
    P, parts = PART[q.dtype]
    dlt = (d * parts + 16) * U * big[..., None]
    floor = FLOOR[q.dtype] + bank.slots * 2.0 ** -126 * 6 * 2.0 ** 8
    if q.dtype != torch.bfloat16:
        # Softmax weights as two fp16 numbers after a factor of 2^12, the row's largest at least 2^12: a weight's error is at most 2^-22 of it (inside
        # 2^-20 * mag) or half of fp16's smallest step, 2^-25 / 2^12 = 2^-37 of the row's largest, which the sum of weights is not below; a slot times
        # its value, of at most 6 * 2^13 (beyond it the products are bf16 ones), the channel's largest by bank head.
        top = values.nan_to_num(0).abs().amax(2).clamp(max=6 * 2.0 ** 13)
        floor = floor + (bank.slots * 2.0 ** -37 * top).repeat_interleave(hq // bank.heads, 1)[:, None]
    _within(got, ref, (HALF[q.dtype] + P) * ref.abs() + (P + 2 * dlt + 2.0 ** -20) * mag + floor)
    if weigh:
        rows = t * hq // bank.heads
        total = base + received
        _within(bank.weight, total, (2 * (d * parts + 16) * U * big.amax() + 2.0 ** -20 + rows * U) * received + 2 * U * total.abs() + rows * 2.0 ** -126)
    else:
        assert torch.equal(bank.weight.double().cpu(), base)
    return got


# batch, heads, group, tokens, slots, lens, dk, dv, causal, count
READ = [
    (1, 1, 1, 1, 1, (1,), 64, 64, False, None),
    (2, 2, 4, 1, 70, (0, 65), 64, 64, False, None),                      # an empty stream
    (3, 2, 3, 1, 300, (63, 64, 257), 128, 128, False, None),
    (1, 3, 8, 2, 1000, (999,), 128, 128, True, None),
    (2, 1, 1, 17, 129, (128, 30), 64, 128, True, (17, 5)),
    (2, 2, 2, 9, 40, (6, 40), 128, 64, True, (9, 0)),                    # more tokens than slots: rows that see nothing; a stream without tokens
    (1, 1, 1, 65, 333, (333,), 128, 512, False, None),
    (2, 1, 5, 40, 513, (513, 200), 256, 256, True, (40, 33)),
    (1, 2, 1, 3, 2100, (2048,), 128, 192, False, None),
    (2, 1, 2, 70, 700, (700, 650), 128, 128, True, (70, 64)),
    (1, 1, 16, 8, 600, (590,), 64, 64, False, None),
]


@pytest.mark.parametrize("weigh", (False, True))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", READ, ids=lambda c: "x".join(map(str, c[:5])) + f"-{c[6]}-{c[7]}")
def test_read(case, dtype, weigh):
    b, h, grp, t, slots, lens, dk, dv, causal, count = case
    bank = _filled(b, h, slots, dk, dv, lens, seed=t)
    bank.weight.copy_(torch.rand(bank.weight.shape, generator=torch.Generator().manual_seed(9)))
    g = torch.Generator().manual_seed(slots)
    q = (2 * torch.randn(b, t, h * grp, dk, generator=g)).to(dtype)
    _check_read(bank, q, causal, None if count is None else torch.tensor(count, dtype=torch.int32), weigh)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_read_peaked_rows_and_scales(dtype):
    """Logits in the hundreds of either sign (one slot takes everything), a scale of its own, keys of very different blocks."""
    bank = _filled(1, 2, 400, 128, 64, (391,), seed=4, spread=6.0)
    g = torch.Generator().manual_seed(2)
    q = (8 * torch.randn(1, 5, 4, 128, generator=g)).to(dtype)
    _check_read(bank, q, False, None, True)
    _check_read(bank, q, True, None, True, scale=-0.7)
    _check_read(bank, q, False, None, False, scale=0.0)


def test_read_strided_queries():
    bank = _filled(2, 2, 100, 64, 64, (100, 77))
    joint = torch.randn(2, 3, 4 * 64 + 5, generator=torch.Generator().manual_seed(3))
    for lo in (0, 5):                                             # aligned heads in unaligned token rows; an odd start
        q = joint[..., lo:lo + 256].view(2, 3, 4, 64)
        _check_read(bank, q, False, None, False, dev_q=_to_dev(q, True))
    q = torch.randn(2, 4, 3, 64, generator=torch.Generator().manual_seed(4))
    _check_read(bank, q.transpose(1, 2), False, None, True, dev_q=q.to(DEV).transpose(1, 2))


def test_read_not_a_number_block():
    """A key block that stands for NaN makes the rows that see it NaN, and no others."""
    bank = _filled(2, 1, 90, 64, 64, (90, 90))
    bank.key_scales[0, 0, 70, 1] = 255
    q = torch.randn(2, 40, 1, 64, generator=torch.Generator().manual_seed(3))
    got = _check_read(bank, q, True, None, False).cpu()
    assert bool(got[0, 20:].isnan().all()) and not bool(got[0, :20].isnan().any()) and not bool(got[1].isnan().any())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dv,tokens", [(64, 20), (64, 90), (128, 20), (256, 90)])
def test_read_not_a_number_values(dv, tokens, dtype):
    """A value block that stands for NaN: its 32 channels are NaN for the rows that see the slot, no others; what no row sees yet may hold anything."""
    bank = _filled(2, 1, 200, 64, dv, (200, 150))
    for b, slot, blk in ((0, 190, dv // 32 - 1), (0, 199, 0), (1, 149 - tokens // 2, 1)):
        bank.value_scales[b, 0, slot, blk] = 255
    q = torch.randn(2, tokens, 1, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    got = _check_read(bank, q, True, None, True).isnan().cpu()
    assert int(got[0, tokens - 10, 0].sum()) == 32 and int(got[0, tokens - 11].sum()) == 0 and int(got[0, -1, 0].sum()) == 64
    assert int(got[1].sum()) == 32 * (tokens - (tokens - 1 - tokens // 2))
    _check_read(bank, q, False, None, False)


def test_read_huge_logits_with_zero_scale_and_split_banks():
    """scale = 0: every slot weighs the same; a bank long enough for many slices, one of them far ahead of the others."""
    bank = _filled(1, 1, 9000, 64, 64, (8999,), spread=30.0)
    for rows in (3, 80):
        q = 100 * torch.randn(1, rows, 1, 64, generator=torch.Generator().manual_seed(3))
        _check_read(bank, q, False, None, True, scale=0.0)
        _check_read(bank, q, True, None, True)


@pytest.mark.parametrize("weigh", (False, True))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("which", ("one key block", "one value block", "all keys", "all values", "small values", "zero blocks"))
def test_read_blocks_of_every_size(which, dtype, weigh):
    """Blocks whose numbers lie far outside fp16 beside ordinary ones, in some slices of the bank and not in others; queries that make their
    logits ordinary again."""
    bank = _filled(2, 1, 2500, 64, 128, (2500, 2049))
    scales, codes, up = {"key": (bank.key_scales, bank.key_codes, 30), "val": (bank.value_scales, bank.value_codes, 90)}["key" if "key" in which else "val"]
    if which.startswith("one"):
        scales[0, 0, 2077, 1] += up
    elif which.startswith("all"):
        scales[:, :, :2049, 1] += up
    elif which.startswith("small"):
        scales[:, :, :2049] -= 80
    else:
        codes[:, :, 100:2000, :16] &= 0x88
        scales[:, :, 100:2000, 0] = 7
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 70, 2, 64, generator=g)
    if up == 30:
        q[..., 32:] *= 2.0 ** -13                       # (fp16 holds them: the block's logits are of 2^17 + 3)
        q[:, ::2, :, 32:] *= 2.0 ** -10
    _check_read(bank, q.to(dtype), False, None, weigh)
    _check_read(bank, q.to(dtype), True, None, weigh)


@pytest.mark.parametrize("up", (-100, -30, 40, 110))
def test_read_queries_of_every_size(up):
    """fp32 queries far outside fp16, the scale undoing it; rows of zeros among them."""
    bank = _filled(1, 2, 700, 128, 64, (690,))
    q = torch.randn(1, 40, 4, 128, generator=torch.Generator().manual_seed(5)) * 2.0 ** (up + torch.arange(40).remainder(11).float()).view(1, 40, 1, 1)
    q[:, 7] = 0
    q[..., 5] *= 2.0 ** -12
    for weigh in (False, True):
        _check_read(bank, q, True, None, weigh, scale=2.0 ** -(up + 8))
        _check_read(bank, q, False, None, weigh, scale=2.0 ** -(up + 8))


@pytest.mark.parametrize("scale", (0.0, 2.0 ** -128, -2.0 ** -128))
def test_read_scales_below_the_normal_numbers(scale):
    """Logits of 2^122 ahead of the scale: a scale of 0 leaves equal weights, a subnormal one (exact in 32 bits) logits of 2^-6; both kernels."""
    bank = _filled(1, 1, 300, 64, 64, (290,))
    for rows in (3, 80):
        q = 2.0 ** 118 * torch.randn(1, rows, 1, 64, generator=torch.Generator().manual_seed(3))
        _check_read(bank, q, True, None, True, scale=scale)
        _check_read(bank, q, False, None, True, scale=scale)


def test_read_same_twice_and_tokens_zero():
    bank = _filled(1, 2, 900, 128, 128, (900,))
    q = torch.randn(1, 33, 8, 128, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    w = []
    for _ in range(3):
        bank.weight.zero_()
        out = ops.bank4_read(bank, q, weigh=True)
        w.append((out, bank.weight.clone()))
    assert all(torch.equal(w[0][0], a) and torch.equal(w[0][1], b) for a, b in w)
    assert ops.bank4_read(bank, q[:, :0], weigh=True).shape == (1, 0, 8, 128) and torch.equal(bank.weight, w[0][1])


def test_read_far_slots_in_a_long_bank():
    """Rows behind 2^31 bytes of keys: 2^25 + 100 slots of 64 bytes of codes; all rows stand for 0 but the last twenty."""
    n = (1 << 25) + 100
    bank = ops.Bank4.empty(1, 1, n, 128, 64, device=DEV)
    for t, v in ((bank.key_codes, 0), (bank.key_scales, 127), (bank.value_codes, 0), (bank.value_scales, 127)):
        t.fill_(v)
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(1, 20, 1, 128, generator=g), torch.randn(1, 20, 1, 64, generator=g)
    ops.bank4_append(bank, k.to(DEV), v.to(DEV), at=torch.tensor([n - 20], dtype=torch.int32, device=DEV))
    q = 12 * torch.randn(1, 2, 1, 128, generator=g)
    got = ops.bank4_read(bank, q.to(DEV), weigh=True).double().cpu()
    kk, vv = (O.unpack(a[0, 0, n - 20:].cpu(), s[0, 0, n - 20:].cpu()) for a, s in ((bank.key_codes, bank.key_scales), (bank.value_codes, bank.value_scales)))
    for t in range(2):
        x = kk @ q[0, t, 0].double() / 128 ** 0.5
        p = torch.exp(x) / (torch.exp(x).sum() + (n - 20))
        assert float((got[0, t, 0] - p @ vv).abs().max()) <= 1e-4 * float((p @ vv.abs()).max())
    last = ops.bank4_values(bank, first=torch.tensor([n - 20], dtype=torch.int32, device=DEV), count=20, dtype=torch.float32)
    assert torch.equal(last[0][0, 0].double().cpu(), kk)
    assert abs(float(bank.weight.double().sum()) - 2) < 1e-3


# batch, heads, slots, lens, keep, first, recent
EVICT = [
    (1, 1, 1, (1,), 1, 0, 0),
    (2, 3, 50, (50, 20), 30, 4, 5),
    (2, 2, 5000, (5000, 4097), 1500, 0, 0),
    (1, 2, 3000, (2999,), 2998, 10, 100),
    (3, 1, 1500, (1500, 0, 700), 600, 300, 300),                   # nothing left to choose
    (1, 1, 20000, (19999,), 12345, 1, 1),
    (2, 1, 32768, (32768, 32767), 8000, 7, 9),
    (1, 1, 45000, (44000,), 30001, 100, 0),                          # more keys than the registers of a workgroup hold
]


def test_evict_wide_rows():
    """Rows of whole dwords of scales (128 / 512 channels): every byte and weight of the kept slots, in order."""
    bank, out = _filled(2, 1, 300, 128, 512, (300, 250)), _dirty(2, 1, 200, 128, 512, seed=3)
    bank.weight.copy_(torch.rand(bank.weight.shape, generator=torch.Generator().manual_seed(1)))
    got = ops.bank4_evict(bank, 190, out, first=3, recent=20).cpu().long()
    assert torch.equal(got.int(), O.evict(bank.weight.cpu(), bank.lens.cpu(), 190, 3, 20)[0])
    for src, dst in ((bank.key_codes, out.key_codes), (bank.key_scales, out.key_scales), (bank.value_codes, out.value_codes),
                     (bank.value_scales, out.value_scales), (bank.weight[..., None], out.weight[..., None])):
        for b in range(2):
            assert torch.equal(dst[b, 0, :190].cpu(), src[b, 0].cpu()[got[b, 0]])


@pytest.mark.parametrize("ties", (False, True))
@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, c[2:])))
def test_evict(case, ties):
    b, h, slots, lens, keep, first, recent = case
    bank = _filled(b, h, slots, 64, 96, lens)
    g = torch.Generator().manual_seed(slots)
    w = torch.rand(bank.weight.shape, generator=g)
    if ties:
        w = torch.floor(w * 4) / 4
        w[..., ::7] = float("nan")
        w[..., 1::5] = -0.0
        w[..., 2::11] = float("inf")
        w[..., 3::11] = -1.5
    bank.weight.copy_(w)
    out = _dirty(b, h, keep + 3, 64, 96, seed=8)
    before = [t.clone().cpu() for t in (out.key_codes, out.key_scales, out.value_codes, out.value_scales, out.weight)]
    got = ops.bank4_evict(bank, keep, out, first=first, recent=recent)
    ref, fresh = O.evict(w, bank.lens.cpu(), keep, first, recent)
    assert torch.equal(got.cpu(), ref) and torch.equal(out.lens.cpu(), fresh)
    for src, dst, old in zip((bank.key_codes, bank.key_scales, bank.value_codes, bank.value_scales, bank.weight),
                             (out.key_codes, out.key_scales, out.value_codes, out.value_scales, out.weight), before):
        src, dst = src.cpu(), dst.cpu()
        want = old.clone()
        for i in range(b):
            for j in range(h):
                n = int(fresh[i])
                want[i, j, :n] = src[i, j, ref[i, j, :n].long()]
        assert torch.equal(dst.view(torch.uint8), want.view(torch.uint8))


# ------------------------------------------------------------------------------------------------ together
def _layer_step(bank, spare, x, pos, plan, wq, wk, keep):
    """One step of a token-memory layer on a frame's joint projection x [B, N, (Hq + 2 Hk) D]: norm + rotary, append, read, evict."""
    b, n, _ = x.shape
    q, k, v = x[..., :256].view(b, n, 4, 64), x[..., 256:384].view(b, n, 2, 64), x[..., 384:].view(b, n, 2, 64)
    q, k = ops.norm_rotary(q, k, wq, wk, pos, plan)
    ops.bank4_append(bank, k, v)
    out = ops.bank4_read(bank, q, causal=True, weigh=True)
    slots = ops.bank4_evict(bank, keep, spare, first=5, recent=n)
    return out, slots


def _layer_setup(seed, frames=4, n=24):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(frames, 2, n, 512, generator=g).bfloat16()
    i = torch.arange(n)
    pos = torch.stack([torch.stack([torch.full((n,), f), i // 6, i % 6], -1).expand(2, n, 3) for f in range(frames)]).to(torch.int32)
    wq, wk = 1 + 0.2 * torch.randn(64, generator=g), 1 + 0.2 * torch.randn(64, generator=g)
    return x, pos, wq, wk


def test_token_memory_layer_over_a_clip():
    """Norm + rotary, append, attention, eviction over a clip of frames, two banks in turn, against the oracle run beside it."""
    frames, n, keep = 4, 24, 40
    x, pos, wq, wk = _layer_setup(0, frames, n)
    plan = ops.RotaryAxes(64, (8, 12, 12), device=DEV)
    banks = [ops.Bank4.empty(2, 2, keep + n, 64, 64, device=DEV) for _ in range(2)]
    for f in range(frames):
        bank, spare = banks[f % 2], banks[1 - f % 2]
        before = bank.weight.double().cpu(), bank.lens.cpu().clone()
        out, slots = _layer_step(bank, spare, x[f].to(DEV), pos[f].to(DEV), plan, wq.to(DEV), wk.to(DEV), keep)
        angle = O.angles(pos[f], (8, 12, 12), 10000.0, False)
        q = O.norm_rotary(x[f][..., :256].double().view(2, n, 4, 64), wq.double(), angle, False, 1e-6).bfloat16()
        keys, values = _rows(bank)
        ref, received, mag, big = O.read(keys, values, bank.lens.cpu(), q.double(), torch.full((2,), n), 64 ** -0.5, True)
        # the kernel's q may round the other way where fp32 and fp64 straddle a border: a step of 2^-7 on single elements of 64
        _within(out, ref, 2.0 ** -7 * ref.abs() + (2.0 ** -8 + 2 * 2.0 ** -7 * big[..., None] / 8) * mag)
        assert bank.lens.tolist() == [int(before[1][0]) + n] * 2
        want, fresh = O.evict(bank.weight.cpu(), bank.lens.cpu(), keep, 5, n)
        assert torch.equal(slots.cpu(), want) and torch.equal(spare.lens.cpu(), fresh)
        old = before[0].clone()
        old[:, :, int(before[1][0]):] = 0
        gained = bank.weight.double().cpu()[:, :, :int(bank.lens[0])].sum(-1) - old.sum(-1)
        assert float((gained - 2 * n).abs().max()) < 1e-3          # every row's weights sum to 1


def test_captured_step_replays_like_eager_calls():
    """append (behind the bank's own length), read with weights and evict captured into one graph and replayed with eager work between,
    and a second graph on other banks captured from the same stream: each equals its eager run."""
    x, pos, wq, wk = (t.to(DEV) for t in _layer_setup(1, 6))
    plan = ops.RotaryAxes(64, (8, 12, 12), device=DEV)
    def fresh():
        return [ops.Bank4.empty(2, 2, 200, 64, 64, device=DEV) for _ in range(2)]
    def snap(bank, spare, out, slots):
        return [t.clone() for t in (out, slots, bank.weight[:, :, :int(bank.lens[0])], bank.lens, spare.lens, spare.weight[:, :, :int(spare.lens[0])],
                                    *ops.bank4_values(bank, dtype=torch.float32), *ops.bank4_values(spare, dtype=torch.float32))]
    eager = []
    for off in (0, 1):
        bank, spare = fresh()
        eager.append([snap(bank, spare, *_layer_step(bank, spare, x[f + off], pos[f + off], plan, wq, wk, 40)) for f in range(5)])
    side = torch.cuda.Stream()
    sets = []
    for off in (0, 1):
        bank, spare = fresh()
        xin, pin = x[0].clone(), pos[0].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _layer_step(bank, spare, xin, pin, plan, wq, wk, 40)
        torch.cuda.current_stream().wait_stream(side)
        bank.lens.zero_()
        bank.weight.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = _layer_step(bank, spare, xin, pin, plan, wq, wk, 40)
        sets.append((graph, bank, spare, xin, pin, got))
    for f in range(5):
        for off, (graph, bank, spare, xin, pin, got) in enumerate(sets):
            xin.copy_(x[f + off])
            pin.copy_(pos[f + off])
        for graph, *_ in sets:
            graph.replay()
        ops.rotary_axes(x[0, :, :, :256].view(2, 24, 4, 64), None, pos[0], plan)       # eager work of the program's own
        torch.cuda.synchronize()
        for off, (graph, bank, spare, xin, pin, got) in enumerate(sets):
            for a, b in zip(snap(bank, spare, *got), eager[off][f]):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """Two programs' banks worked on from two streams at the same time: each as alone."""
    x, pos, wq, wk = (t.to(DEV) for t in _layer_setup(2))
    plan = ops.RotaryAxes(64, (8, 12, 12), device=DEV)
    def run(streams):
        banks = [[ops.Bank4.empty(2, 2, 100, 64, 64, device=DEV) for _ in range(2)] for _ in range(2)]
        torch.cuda.synchronize()
        outs = [[], []]
        for f in range(3):
            for i in (0, 1):
                with torch.cuda.stream(streams[i]):
                    outs[i].append(_layer_step(banks[i][f % 2], banks[i][1 - f % 2], x[f + i], pos[f + i], plan, wq, wk, 40))
        torch.cuda.synchronize()
        return outs
    now = torch.cuda.current_stream()
    alone, both = run([now, now]), run([torch.cuda.Stream(), torch.cuda.Stream()])
    for a, b in zip(alone, both):
        for u, v in zip(a, b):
            assert torch.equal(u[0], v[0]) and torch.equal(u[1], v[1])


# ------------------------------------------------------------------------------------------------ padded tokens
# tokens, query heads a bank head, valid tokens of the two streams: rows of one 16-row tile, of two, and of the 128-row kernel
PADDED = [(5, 1, (3, 5)), (2, 3, (1, 0)), (4, 8, (2, 3)), (40, 2, (33, 1))]


@pytest.mark.parametrize("weigh", (False, True))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("slots", (100, 1000, 5000))
@pytest.mark.parametrize("case", PADDED, ids=lambda c: f"{c[0]}x{c[1]}")
def test_read_padded_tokens_are_zero(case, slots, dtype, weigh):
    """Tokens behind a stream's count beside valid ones, over one slice of the bank and several: exactly 0, whatever the bank holds."""
    tokens, group, counts = case
    bank = _filled(2, 2, slots, 64, 128, (slots - 3, slots * 2 // 3), seed=tokens)
    q = 2 * torch.randn(2, tokens, 2 * group, 64, generator=torch.Generator().manual_seed(slots))
    count = torch.tensor(counts, dtype=torch.int32)
    for nan in (False, True):
        if nan:                                                    # a key block that only the valid rows of the first stream meet
            bank.key_scales[0, :, 7, 1] = 255
        for causal in (False, True):
            got = _check_read(bank, q.to(dtype), causal, count, weigh and not nan)
            for b in range(2):
                assert not bool(got[b, counts[b]:].view(torch.uint8).any())
                assert bool(got[b, :counts[b]].isnan().all()) == (nan and b == 0) or not counts[b]


# ------------------------------------------------------------------------------------------------ precision of the products
@pytest.mark.parametrize("tokens,p,floor", [(8, 2.0 ** -16, 0.0), (33, 2.0 ** -11, 2.0 ** -33), (150, 2.0 ** -11, 2.0 ** -33)])
@pytest.mark.parametrize("lens", ((2, 3), (5, 70)))
def test_read_bf16_queries_keep_their_weights(lens, tokens, p, floor):
    """Few slots of near weights and values of either sign, so that an output is far below its terms and shows how its weights were rounded: two
    bf16 numbers (2^-16 of each) with up to 32 rows, one fp16 number (half a step: 2^-11 of each, or 2^-25 / 2^8 of the row's largest) with more."""
    bank = _filled(2, 1, 80, 64, 128, lens, seed=tokens)
    keys, values = _rows(bank)
    q = (0.4 * torch.randn(2, tokens, 1, 64, generator=torch.Generator().manual_seed(6))).bfloat16()
    for causal in (False, True):
        ref, _, mag, big = O.read(keys, values, bank.lens.cpu(), q.double(), torch.full((2,), tokens), 64 ** -0.5, causal)
        got = ops.bank4_read(bank, q.to(DEV), causal=causal)
        tol = (2.0 ** -8 + p) * ref.abs() + (p + 2 * (64 + 16) * U * big[..., None] + 2.0 ** -20) * mag
        _within(got, ref, tol + 80 * (floor * values.nan_to_num(0).abs().amax((1, 2))[:, None, None] + 2.0 ** -126 * 6 * 2.0 ** 8))


@pytest.mark.parametrize("weigh", (False, True))
@pytest.mark.parametrize("which", ("blocks", "silent channel"))
def test_read_fp32_queries_of_far_apart_channels(which, weigh):
    """fp32 rows whose largest channels meet the smallest keys, or keys of 0, and whose logits come from channels 2^30 below: held to 24 bits all the same."""
    bank = _filled(2, 1, 700, 64, 64, (700, 333))
    q = torch.randn(2, 70, 2, 64, generator=torch.Generator().manual_seed(8))
    if which == "blocks":
        bank.key_scales[..., 0], bank.key_scales[..., 1] = 104, 140
        q[..., 32:] *= 2.0 ** -30
        scale = 2.0 ** 15
    else:
        bank.key_codes[..., 2] &= 0x0f                             # channel 5
        q[..., 5] = 2.0 ** 32
        scale = None
    for causal in (False, True):
        _check_read(bank, q, causal, None, weigh, scale=scale)


def _check_many(bank, q, causal, weigh, scale):
    """_check_read for 33 rows and more, with what these hold of a bf16 row's softmax weights: an fp16 number after a factor of 2^8, the row's largest at
    least 2^8, so 2^-11 of each, or half of fp16's smallest step, 2^-25 / 2^8 = 2^-33 of the row's largest (a slot, times the channel's largest value)."""
    if q.dtype != torch.bfloat16:
        return _check_read(bank, q, causal, None, weigh, scale=scale)
    keys, values = _rows(bank)
    d, t = q.shape[3], q.shape[1]
    ref, received, mag, big = O.read(keys, values, bank.lens.cpu(), q.double(), torch.full((q.shape[0],), t), scale or d ** -0.5, causal)
    base = bank.weight.double().cpu()
    got = ops.bank4_read(bank, q.to(DEV), scale=scale, causal=causal, weigh=weigh)
    top = values.nan_to_num(0).abs().amax(2).clamp(max=6 * 2.0 ** 13).repeat_interleave(q.shape[2] // bank.heads, 1)[:, None]
    dlt = (d + 16) * U * big[..., None]
    _within(got, ref, (HALF[q.dtype] + 2.0 ** -11) * ref.abs() + (2.0 ** -11 + 2 * dlt + 2.0 ** -20) * mag + bank.slots * (2.0 ** -33 * top + 2.0 ** -126 * 6 * 2.0 ** 8))
    rows = t * q.shape[2] // bank.heads
    total = base + received if weigh else base
    _within(bank.weight, total, (2 * (d + 16) * U * big.amax() + 2.0 ** -20 + rows * U) * received + 2 * U * total.abs() + rows * 2.0 ** -126)
    return got


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens", (10, 90))
def test_read_blocks_that_append_marked(tokens, dtype):
    """Keys and values with infinities and NaN as append writes them (codes 0 under the scale byte 255): NaN for the rows that see them, and no others."""
    bank = _filled(2, 1, 300, 64, 128, (300, 250))
    g = torch.Generator().manual_seed(tokens)
    k, v = torch.randn(2, 1, 1, 64, generator=g), torch.randn(2, 1, 1, 128, generator=g)
    v[0, 0, 0, 40], k[1, 0, 0, 3] = float("inf"), float("nan")
    lens = bank.lens.clone()
    ops.bank4_append(bank, k.to(DEV), v.to(DEV), at=lens - 5)
    bank.lens.copy_(lens)
    assert int(bank.value_scales[0, 0, 295, 1]) == 255 and not bool(bank.value_codes[0, 0, 295, 16:32].any()) and int(bank.key_scales[1, 0, 245, 0]) == 255
    q = torch.randn(2, tokens, 2, 64, generator=g).to(dtype)
    for causal, seeing in ((True, 5), (False, tokens)):
        got = _check_read(bank, q, causal, None, False).isnan()
        assert bool(got[0, -seeing:, :, 32:64].all()) and int(got[0].sum()) == seeing * 2 * 32
        assert bool(got[1, -seeing:].all()) and int(got[1].sum()) == seeing * 2 * 128
    ops.bank4_read(bank, q.to(DEV), causal=True, weigh=True)       # the first stream's keys are numbers, so its weights are; the other's are NaN
    keys, values = _rows(bank)
    _, ref, _, big = O.read(keys, values, bank.lens.cpu(), q.double(), torch.full((2,), tokens), 64 ** -0.5, True)
    d = (64 * PART[dtype][1] + 16) * U * big[0].max()
    _within(bank.weight[0], ref[0], (2 * d + 2.0 ** -20 + 2 * tokens * U) * ref[0] + 2 * tokens * 2.0 ** -126)
    assert torch.equal(bank.weight[1].isnan().cpu(), ref[1].isnan())


@pytest.mark.parametrize("weigh", (False, True))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("which", ("keys", "values"))
def test_read_smallest_blocks_that_fp16_holds(which, dtype, weigh):
    """Scale bytes 104 .. 112 and their neighbours below: codes of 2^-24 and up, subnormal in fp16."""
    bank = _filled(2, 1, 700, 64, 128, (700, 333))
    scales = bank.key_scales if which == "keys" else bank.value_scales
    for lowest in (104, 102):
        scales.copy_((lowest + torch.arange(scales.numel()) % 9).view(scales.shape))
        q = 2 * torch.randn(2, 70, 2, 64, generator=torch.Generator().manual_seed(8))
        for causal in (False, True):
            _check_many(bank, q.to(dtype), causal, weigh, 2.0 ** 15 if which == "keys" else None)


# ------------------------------------------------------------------------------------------------ angles
def test_rotary_angles_are_rounded_not_cut():
    """Angles next to whole multiples of 2^-32 turns: off by half of that (and 2^-34 for the frequency), so the sine of a small one is off by
    2 pi (2^-33 + 2^-34) and 2^-21 of itself (sine 4u, product u, frequency's double precision none)."""
    for dim in (4, 16):                                            # a wave a row; 16 channels a lane
        pairs, r = dim // 2, 0.8
        base = (2 * math.pi * r * 2.0 ** -32) ** -pairs            # the second pair turns by r 2^-32 turns a position
        plan = ops.RotaryAxes(dim, (pairs,), base=base, device=DEV)
        pos = torch.arange(-9, 10, dtype=torch.int32)
        x = torch.zeros(1, 19, 1, dim)
        x[..., 1] = 1
        for sign, call in ((1, ops.rotary_axes), (-1, ops.rotary_axes_grad)):
            y = call(x.to(DEV), None, pos.to(DEV).view(1, 19, 1), plan)[0]
            ref = sign * torch.sin(pos.double() * 2 * math.pi * r * 2.0 ** -32)
            got = y[0, :, 0, 1 + pairs].double().cpu()
            assert bool(((got - ref).abs() <= 2 * math.pi * (2.0 ** -33 + 2.0 ** -34) + 2.0 ** -21 * ref.abs()).all()), (dim, sign, got, ref)


@pytest.mark.parametrize("weigh", (False, True))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dk,dv,slots", [(128, 512, 2500), (64, 192, 90), (256, 256, 1300)])
def test_read_blocks_outside_fp16_in_some_channels(dk, dv, slots, dtype, weigh):
    """Value blocks outside fp16 in some of a row's channels: the workgroups of those channels run on other numbers than those of the rest, over one slice
    or several, and the rows' slices are joined all the same."""
    bank = _filled(2, 1, slots, dk, dv, (slots, slots - 20))
    bank.value_scales[0, 0, 5, 0] = 150
    bank.value_scales[1, 0, slots // 2, dv // 32 - 1] = 80
    q = 2 * torch.randn(2, 50, 2, dk, generator=torch.Generator().manual_seed(8))
    for causal in (False, True):
        _check_many(bank, q.to(dtype), causal, weigh, None)
