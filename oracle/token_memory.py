"""fp64 restatement of the token-memory operators (rotary positions over several axes, norm + rotary, the 4-bit bank), by their
definitions and without the package's code: what tests/test_gpu_token_memory.py holds the kernels to."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def angles(positions, sections, base, shared):
    """fp64 angle of every pair, [B, N, pairs]."""
    out, i, total = [], 0, sum(sections)
    for a, n in enumerate(sections):
        for j in range(n):
            out.append(positions[..., a].double() * float(base) ** (-(i / total if shared else j / n)))
            i += 1
    return torch.stack(out, -1)


def turn(x, angle, interleaved):
    """x [B, N, H, D] fp64, angle [B, N, pairs]."""
    p = angle.shape[-1]
    u = torch.arange(p) * 2 if interleaved else torch.arange(p)
    v = u + 1 if interleaved else u + p
    c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    y = x.clone()
    y[..., u], y[..., v] = x[..., u] * c - x[..., v] * s, x[..., v] * c + x[..., u] * s
    return y


def norm(x, weight, eps):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight


def norm_rotary(x, weight, angle, interleaved, eps):
    return turn(norm(x, weight, eps), angle, interleaved)


def norm_rotary_grad(dy, x, weight, angle, interleaved, eps):
    """(dx, dweight) by the formula."""
    g = turn(dy, -angle, interleaved)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    wg = g * weight
    return r * (wg - x * r * r * (wg * x).mean(-1, keepdim=True)), (g * x * r).sum((0, 1, 2))


def block_exponents(x):
    """The smallest e in [-120, 125] with max |x| <= 6 * 2^e for every block of 32 channels (python integers of exact comparisons)."""
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1)
    e = torch.full(top.shape, -120, dtype=torch.int64)
    for k in range(-120, 125):
        e[top > 6 * 2.0 ** k] = k + 1
    return e


def quantise(x):
    """fp64 [..., D] -> (codes [..., D] as integers 0..15, scale bytes [..., D / 32]); nearest grid point, ties to the even code."""
    bad = ~torch.isfinite(x.unflatten(-1, (-1, 32))).all(-1)
    x = torch.where(bad.repeat_interleave(32, -1), torch.zeros_like(x), x)
    e = block_exponents(x)
    a = x.abs() * torch.exp2(-e.double()).repeat_interleave(32, -1)
    away = (a[..., None] - GRID).abs()
    best = away.amin(-1, keepdim=True)
    near = away == best                                         # one grid point, or two at the same distance
    code = torch.where(near.sum(-1) == 2, (near * (torch.arange(8) % 2 == 0) * torch.arange(8)).amax(-1), near.int().argmax(-1))
    code = torch.where(bad.repeat_interleave(32, -1), torch.zeros_like(code), code + 8 * torch.signbit(x).long())
    return code, torch.where(bad, torch.full_like(e, 255), e + 127)


def pack(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)


def unpack(codes, scales):
    """Packed uint8 codes and scales -> fp64 values (scale byte 255: NaN)."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = GRID[c & 7] * (1 - 2 * (c >> 3)).double()
    s = torch.where(scales == 255, torch.full(scales.shape, math.nan, dtype=torch.float64), torch.exp2(scales.double() - 127))
    return v * s.repeat_interleave(32, -1)


def read(keys, values, lens, q, count, scale, causal):
    """keys [B, H, S, Dk], values [B, H, S, Dv], q [B, T, Hq, Dk] fp64 -> (out [B, T, Hq, Dv], received [B, H, S], sum of p |v| [B, T, Hq, Dv],
    largest sum |q| |k| [B, T, Hq])."""
    b, t, hq, _ = q.shape
    h, s = keys.shape[1], keys.shape[2]
    out = torch.zeros(b, t, hq, values.shape[3], dtype=torch.float64)
    mag, big = out.clone(), torch.zeros(b, t, hq, dtype=torch.float64)
    received = torch.zeros(b, h, s, dtype=torch.float64)
    for i in range(b):
        n = max(0, min(int(lens[i]), s))
        c = max(0, min(int(count[i]), t))
        for j in range(hq):
            k, v = keys[i, j * h // hq], values[i, j * h // hq]
            for u in range(c):
                m = max(0, n - c + u + 1) if causal else n
                if m == 0:
                    continue
                x = k[:m] @ q[i, u, j] * scale
                p = torch.softmax(x, 0)
                out[i, u, j], mag[i, u, j] = p @ v[:m], p @ v[:m].abs()
                big[i, u, j] = (k[:m].abs() @ q[i, u, j].abs()).max() * abs(scale)
                received[i, j * h // hq, :m] += p
    return out, received, mag, big


def evict(weight, lens, keep, first, recent):
    """Kept slots [B, H, keep] (-1 behind) and the new lengths."""
    b, h, s = weight.shape
    slots = torch.full((b, h, keep), -1, dtype=torch.int32)
    fresh = []
    for i in range(b):
        n = max(0, min(int(lens[i]), s))
        fresh.append(min(n, keep))
        for j in range(h):
            kept = list(range(n))
            if n > keep:
                w = [-math.inf if math.isnan(v) else v for v in weight[i, j, :n].tolist()]
                nan = [math.isnan(v) for v in weight[i, j, :n].tolist()]
                free = sorted(range(first, n - recent), key=lambda x: (nan[x], -w[x], x))
                kept = sorted(list(range(first)) + free[:keep - first - recent] + list(range(n - recent, n)))
            slots[i, j, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
    return slots, torch.tensor(fresh, dtype=torch.int32)
