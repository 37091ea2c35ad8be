"""Microscaled 4-bit floating point in plain float64 on the CPU: what codes and exponents stand for, the quantiser, and products with the
bound on how far a float32 sum may be from them."""
import torch

VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def numbers(data, exponents):
    """data [rows, K / 2], exponents [rows, K / 32] uint8 -> float64 [rows, K]"""
    data, exponents = data.cpu(), exponents.cpu()
    code = torch.stack([data & 15, data >> 4], -1).reshape(data.shape[0], -1, 32)
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64), exponents.double() - 127)
    power = torch.where(exponents == 255, torch.tensor(float("nan"), dtype=torch.float64), power)
    return (VALUES[code.long()] * power[..., None]).reshape(data.shape[0], -1)


def of(w):
    """An ``ops.Mxfp4`` matrix, or a stack of them, as float64."""
    e = w.exponents()
    if w.data.dim() == 3:
        return torch.stack([numbers(d, x) for d, x in zip(w.data, e)])
    return numbers(w.data, e)


def rounded(x):
    """Rows of x [rows, K] as the format holds them, by nearest neighbour among the eight magnitudes: (float64 [rows, K], exponents)."""
    x = x.cpu().double().reshape(x.shape[0], -1, 32)
    largest = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    safe = torch.where(fine, largest, torch.ones_like(largest))
    _, up = torch.frexp(safe)                                   # safe < 2 ** up, at least half of it
    e = torch.where(safe == 0, torch.zeros_like(up), (up - 1 - 2 + 127).clamp_min(0))
    y = x.abs() * torch.pow(torch.tensor(2.0, dtype=torch.float64), (127 - e).double())[..., None]
    mag = VALUES[:8]
    gap = (torch.where(fine[..., None], y, torch.zeros_like(y)).clamp_max(6.0)[..., None] - mag).abs()
    best = gap.amin(-1, keepdim=True)
    tied = gap == best                                          # one or two neighbours
    even = torch.arange(8) % 2 == 0
    code = torch.where(tied.sum(-1) > 1, (tied & even).double().argmax(-1), tied.double().argmax(-1))
    value = mag[code] * torch.where(x < 0, -1.0, 1.0) * torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 127).double())[..., None]
    value = torch.where(fine[..., None], value, torch.tensor(float("nan"), dtype=torch.float64))
    return value.reshape(x.shape[0], -1), torch.where(fine, e, torch.tensor(255)).to(torch.uint8)


def product(x, w):
    """(x w^T, how far a result may be off before it is rounded to the output type), float64.

    Products of the operands are exact in float32.  A tensor-core accumulator takes 16 of them at a time and cuts each sum to 24 bits or more: at
    most 2^-23 of a partial sum's bound for each of K / 16 steps, as much again for aligning the terms of a step, and 32 additions of partial sums
    of shares of K.  Partial sums are bounded by sum |x| |w|.  (Float32 sums below 2^-126 have a step of 2^-149.)"""
    x, w = x.double().cpu(), w.double().cpu()
    size = x.abs() @ w.abs().T
    return x @ w.T, size * (2 * x.shape[1] / 16 + 32) * 2.0 ** -23 + 2.0 ** -140


def check(got, want, slack):
    """got within slack of want, plus half a step of its type."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[got.dtype]
    got = got.double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    allowed = slack + half * (want.abs() + slack)
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert not torch.isnan(got).any() and worst <= 1.0, f"{worst:.3g} of what rounding allows, at {(off / allowed).argmax().item()}"
    return worst


def random_exponents(rows, k, g, low=110, high=130):
    return torch.randint(low, high + 1, (rows, k // 32), generator=g, dtype=torch.uint8)


def random_matrix(rows, k, g, low=115, high=125):
    """Any codes, exponents of a few binades: (data, exponents) on the CPU."""
    return torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8), random_exponents(rows, k, g, low, high)
