"""Token-memory operators without a GPU: the fp64 oracle against itself (gradients against differences, the 4-bit grid), the rotary
plan's frequencies, and every refusal of the entry points."""
import math

import pytest
import torch

from mivos_amd import _lib, ops
from mivos_amd._lib import MivosHipError
from oracle import token_memory as O


def test_rotary_plan_frequencies_are_exact_fractions_of_a_turn():
    for sections, shared, base in (((8, 12, 12), False, 10000.0), ((5, 0, 9), True, 500000.0), ((1,), False, 0.5)):
        plan = ops.RotaryAxes(2 * sum(sections) + 4, sections, base=base, shared=shared, device="cpu")
        i = 0
        for a, n in enumerate(sections):
            for j in range(n):
                f = base ** -(i / sum(sections) if shared else j / n) / (2 * math.pi)
                got = (int(plan.freq[i]) % 2 ** 64) / 2 ** 64
                assert abs(got - f % 1) < 1e-15 * max(1, f) and int(plan.axis[i]) == a
                i += 1
        assert plan.pairs == i


def test_oracle_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(2, 3, 2, 24, generator=g, dtype=torch.float64), torch.randn(2, 3, 2, 24, generator=g, dtype=torch.float64)
    w = 1 + 0.3 * torch.randn(24, generator=g, dtype=torch.float64)
    angle = O.angles(torch.randint(-50, 50, (2, 3, 2), generator=g), (4, 5), 100.0, False)
    for inter in (False, True):
        dx, dw = O.norm_rotary_grad(dy, x, w, angle, inter, 1e-3)
        f = lambda x, w: (O.norm_rotary(x, w, angle, inter, 1e-3) * dy).sum()  # noqa: E731
        for _ in range(5):
            u, v = torch.randn(x.shape, generator=g, dtype=torch.float64), torch.randn(24, generator=g, dtype=torch.float64)
            h = 1e-5
            slope = (f(x + h * u, w + h * v) - f(x - h * u, w - h * v)) / (2 * h)
            assert abs(slope - (dx * u).sum() - (dw * v).sum()) < 1e-7 * (1 + abs(slope))


def test_four_bit_grid():
    """The nearest grid point of the smallest scale that holds the block; ties to the even code; infinities and NaN."""
    x = torch.zeros(1, 64, dtype=torch.float64)
    x[0, :12] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 0.2500001, -6], dtype=torch.float64)
    x[0, 32] = 6.0001
    code, scale = O.quantise(x)
    assert code[0, :12].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8, 14, 1, 15] and scale.tolist() == [[127, 128]]
    x[0, 40] = math.nan
    code, scale = O.quantise(x)
    assert scale.tolist() == [[127, 255]] and bool(O.unpack(O.pack(code), scale)[0, 32:].isnan().all())
    tiny, huge = torch.full((1, 32), 2.0 ** -140, dtype=torch.float64), torch.full((1, 32), 3.4e38, dtype=torch.float64)
    assert O.quantise(tiny)[1].item() == 7 and O.quantise(huge)[1].item() == 252


def _bank(**kw):
    a = dict(batch=2, heads=2, slots=16, key_dim=64, value_dim=64)
    a.update(kw)
    return ops.Bank4.empty(**a, device="cpu")


def _raises(match, fn, *args, **kw):
    with pytest.raises(MivosHipError, match=match):
        fn(*args, **kw)


def test_rotary_refusals():
    plan = ops.RotaryAxes(32, (4, 6, 6), device="cpu")
    q, pos, w = torch.zeros(2, 3, 4, 32), torch.zeros(2, 3, 3, dtype=torch.int32), torch.ones(32)
    _raises("do not fit", ops.RotaryAxes, 32, (9, 9), device="cpu")
    _raises("do not fit", ops.RotaryAxes, 600, (9, 9), device="cpu")
    _raises("do not fit", ops.RotaryAxes, 32, (), device="cpu")
    _raises("base", ops.RotaryAxes, 32, (4,), base=0.0, device="cpu")
    _raises("expected", ops.rotary_axes, q[0], None, pos, plan)
    _raises("channels", ops.rotary_axes, torch.zeros(2, 3, 4, 34), None, pos, plan)
    _raises("channel stride", ops.rotary_axes, torch.zeros(2, 3, 32, 4).transpose(2, 3), None, pos, plan)
    _raises("expected", ops.rotary_axes, q, torch.zeros(2, 2, 4, 32), pos, plan)
    _raises("k is", ops.rotary_axes, q, q.half(), pos, plan)
    _raises("positions", ops.rotary_axes, q, None, pos.long(), plan)
    _raises("positions", ops.rotary_axes, q, None, pos[..., :2], plan)
    _raises("float32, float16 or bfloat16", ops.rotary_axes, q.double(), None, pos, plan)
    _raises("eps", ops.norm_rotary, q, None, w, None, pos, plan, eps=-1.0)
    _raises("eps", ops.norm_rotary, q, None, w, None, pos, plan, eps=math.nan)
    _raises("q_weight", ops.norm_rotary, q, None, w.half(), None, pos, plan)
    _raises("k_weight", ops.norm_rotary, q, q, w, None, pos, plan)
    _raises("dk goes with k", ops.norm_rotary_grad, q, None, q, q, w, w, pos, plan)
    _raises("expected", ops.norm_rotary_grad, q[:1], None, q, None, w, None, pos, plan)
    _raises("its gradient", ops.norm_rotary_grad, q.half(), None, q, None, w, None, pos, plan)
    for call in (lambda: ops.rotary_axes(q, None, pos, plan), lambda: ops.norm_rotary(q, q, w, w, pos, plan),
                 lambda: ops.norm_rotary_grad(q, q, q, q, w, w, pos, plan)):
        _raises("no CPU fallback", call)


def test_bank_refusals():
    _raises("channels", ops.Bank4.empty, 1, 1, 4, 48, 64, device="cpu")
    _raises("streams", ops.Bank4.empty, 0, 1, 4, 64, 64, device="cpu")
    b = _bank()
    parts = (b.key_codes, b.key_scales, b.value_codes, b.value_scales, b.weight, b.lens)
    _raises("dense", ops.Bank4, *parts[:4], b.weight.double(), b.lens)
    _raises("dense", ops.Bank4, *parts[:5], b.lens.long())
    _raises("dense", ops.Bank4, b.key_codes[:, :, ::2], *parts[1:])
    _raises("share memory", ops.Bank4, b.key_codes, b.key_scales, b.key_codes, *parts[3:])
    off = torch.zeros(b.key_codes.numel() + 8, dtype=torch.uint8)[8:].view(b.key_codes.shape)
    _raises("aligned", ops.Bank4, off, *parts[1:])
    k, at = torch.zeros(2, 3, 2, 64), torch.zeros(2, dtype=torch.int32)
    _raises("keys", ops.bank4_append, b, k[:, :, :1], k)
    _raises("values", ops.bank4_append, b, k, k[:, :2])
    _raises("values", ops.bank4_append, b, k, k.half())
    _raises("channel stride", ops.bank4_append, b, torch.zeros(2, 3, 64, 2).transpose(2, 3), k)
    _raises("at", ops.bank4_append, b, k, k, at=at.long())
    _raises("at", ops.bank4_append, b, k, k, at=at[:1])
    _raises("overlaps", ops.bank4_append, b, k, k, count=b.lens)
    _raises("got", ops.bank4_append, b, k.double(), k.double())
    _raises("slots", ops.bank4_values, b, count=17)
    _raises("float32 or bfloat16", ops.bank4_values, b, dtype=torch.float16)
    _raises("query heads", ops.bank4_read, b, torch.zeros(2, 1, 3, 64))
    _raises("queries", ops.bank4_read, b, torch.zeros(1, 1, 2, 64))
    _raises("count", ops.bank4_read, b, torch.zeros(2, 1, 2, 64), count=at[:1])
    _raises("keys of 96", ops.bank4_read, _bank(key_dim=96), torch.zeros(2, 1, 2, 96))
    _raises("values of 96", ops.bank4_read, _bank(value_dim=96), torch.zeros(2, 1, 2, 64))
    o = _bank(slots=8)
    _raises("share memory", ops.bank4_evict, b, 8, b)
    _raises("differ", ops.bank4_evict, b, 8, _bank(heads=1))
    for keep, first, recent in ((0, 0, 0), (9, 0, 0), (8, 5, 4), (8, -1, 0), (8, 0, -1)):
        _raises("keep", ops.bank4_evict, b, keep, o, first=first, recent=recent)
    for call in (lambda: ops.bank4_append(b, k, k), lambda: ops.bank4_values(b), lambda: ops.bank4_read(b, torch.zeros(2, 1, 2, 64)),
                 lambda: ops.bank4_evict(b, 8, o)):
        _raises("no CPU fallback", call)


def test_bank_buffers_are_fixed_and_may_come_from_one_allocation():
    b = _bank()
    _raises("fixed", setattr, b, "lens", torch.zeros(2, dtype=torch.int32))
    lens = b.lens
    b.lens += 3                                                      # writes into the buffer
    assert b.lens is lens and lens.tolist() == [3, 3]
    whole = torch.zeros(2, 2, 2, 16, 32, dtype=torch.uint8)          # codes of keys and values side by side
    c = ops.Bank4(whole[0], b.key_scales, whole[1], b.value_scales, b.weight, b.lens)
    _raises("share memory", ops.bank4_evict, b, 8, c)
    _raises("share memory", ops.Bank4, whole[0], b.key_scales, whole[0], b.value_scales, b.weight, b.lens)
    for scale in (math.inf, math.nan, 2e38, -2e38):
        _raises("scale", ops.bank4_read, b, torch.zeros(2, 1, 2, 64), scale=scale)


def test_c_entries_check_their_arguments_without_a_gpu():
    """The C ABI's own checks (a caller other than the Python wrappers): status codes, no launch."""
    import ctypes as C
    lib = _lib.load()
    b = _bank()
    d = b._desc
    assert lib.mivos_bank4_read_workspace_bytes(d, 3, 1, 0, 0) == -1 and b"query heads" in lib.mivos_last_error()
    assert lib.mivos_bank4_read_workspace_bytes(d, 4, 5, 0, 1) >= 2 * 2 * 10 * 64 * 4
    assert lib.mivos_bank4_read_workspace_bytes(None, 4, 5, 0, 1) == -1
    assert lib.mivos_bank4_read(d, 1, 0, 0, 0, 0, 4, 5, None, 1.0, 0, 1, 1, None, 0, None) == -1 and b"workspace" in lib.mivos_last_error()
    assert lib.mivos_bank4_append(d, None, 0, 0, 0, None, 0, 0, 0, 0, None, None, 1, None) == -1
    assert lib.mivos_bank4_append(d, 1, 0, 0, 0, 1, 0, 0, 0, 7, 1, None, 1, None) == -1
    assert lib.mivos_bank4_values(d, None, 17, 1, 1, 0, None) == -1 and lib.mivos_bank4_values(d, None, 1, 1, 1, 1, None) == -1
    assert lib.mivos_bank4_evict(d, d, 4, 0, 0, 1, None) == -1 and b"share memory" in lib.mivos_last_error()
    bad = _lib.Bank4Desc(*(getattr(d, n) for n, _ in d._fields_))
    bad.key_dim = 48
    assert lib.mivos_bank4_values(bad, None, 1, 1, 1, 0, None) == -1
    r = _lib.RotaryDesc()
    assert lib.mivos_rotary_axes(r, None) == -1 and lib.mivos_rotary_axes(None, None) == -1
    r.dim, r.pairs, r.batch, r.tokens, r.freq, r.axis = 32, 17, 1, 1, 1, 1
    assert lib.mivos_rotary_axes(r, None) == -1
    r.pairs = 16
    assert lib.mivos_rotary_axes(r, None) == -1 and b"positions" in lib.mivos_last_error()
    assert lib.mivos_norm_rotary_grad(r, None, None, None) == -1
    assert C.sizeof(_lib.RotaryRows) == 88 and C.sizeof(_lib.Bank4Desc) == 80
    assert C.sizeof(_lib.RotaryDesc) == ops._ROTARY.size and _lib.RotaryDesc.eps.offset + 4 == ops._ROTARY.size


def test_c_entries_refuse_overlapping_and_unaligned_buffers():
    """What the Python wrappers refuse, the C entries refuse too: counts on top of the lengths that append writes, a bank that shares any of its
    seven buffers with the one it is brought down from, codes and scales off 16 bytes."""
    lib = _lib.load()
    b, o = _bank(), _bank(slots=8)
    d = b._desc
    copy = lambda s: _lib.Bank4Desc(*(getattr(s, n) for n, _ in s._fields_))  # noqa: E731
    append = lambda desc, at, count: lib.mivos_bank4_append(desc, 16, 0, 0, 0, 16, 0, 0, 0, 0, at, count, 3, None)  # noqa: E731
    for at, count in ((d.lens + 4, None), (d.lens - 4, None), (64, d.lens), (64, d.lens + 4), (d.lens, d.lens - 4), (d.lens, d.lens)):
        assert append(d, at, count) == -1 and b"overlap" in lib.mivos_last_error(), (at - d.lens, count)
    last = {"key_codes": 2 * 2 * 16 * 32, "key_scales": 2 * 2 * 16 * 2, "value_codes": 2 * 2 * 16 * 32, "value_scales": 2 * 2 * 16 * 2, "weight": 2 * 2 * 16 * 4, "lens": 8,
            "status": 12}
    for name, size in last.items():
        for at in (getattr(d, name), getattr(d, name) + (size - 16 if size > 16 else size - 4)):
            c = copy(o._desc)
            setattr(c, name, at)
            assert lib.mivos_bank4_evict(d, c, 4, 0, 0, 64, None) == -1 and b"share memory" in lib.mivos_last_error(), name
    c = copy(o._desc)
    c.value_codes = d.weight                                       # one buffer of the one, another of the other
    assert lib.mivos_bank4_evict(d, c, 4, 0, 0, 64, None) == -1 and b"share memory" in lib.mivos_last_error()
    for name in ("key_codes", "key_scales", "value_codes", "value_scales"):
        c = copy(d)
        setattr(c, name, getattr(d, name) + 8)
        assert append(c, d.lens, None) == -1 and b"aligned" in lib.mivos_last_error(), name
        assert lib.mivos_bank4_values(c, None, 1, 16, 16, 0, None) == -1 and lib.mivos_bank4_read_workspace_bytes(c, 4, 5, 0, 1) == -1


def test_rotary_plan_bases_at_the_limits():
    """Frequencies of the smallest base against exact fractions, and the bases below it, whose fractions of a turn 50 digits do not hold."""
    from fractions import Fraction
    pi = Fraction(31415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679, 10 ** 100)
    plan = ops.RotaryAxes(8, (2, 1, 1), base=2.0 ** -96, device="cpu")      # the second pair: 2^48
    turn = Fraction(2 ** 64) / (2 * pi)
    for i, f in ((0, 1), (1, 2 ** 48), (2, 1), (3, 1)):
        away = (int(plan.freq[i]) - turn * f) % 2 ** 64
        assert min(away, 2 ** 64 - away) <= 1
    for base in (1e-31, 5e-324, 0.0, -1.0, math.inf, math.nan):
        _raises("base", ops.RotaryAxes, 8, (4,), base=base, device="cpu")
