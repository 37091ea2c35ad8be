"""Operators on microscaled 4-bit weights, as cases that can be timed and compared: matrices held as MXFP4 (4-bit floating-point numbers of one
sign, two exponent and one mantissa bit, in blocks of 32 along a row that share a power of two), quantising rows to it, reading rows back (the
lookup in a 4-bit embedding table), and the contractions of a decoder with such weights - bfloat16 activations on 4-bit weights, 4-bit activations
on 4-bit weights, and rows grouped by expert on a stack of 4-bit weights.

Layout.  ``data`` [rows, K / 2] uint8: number 2 i of a row in the low half of byte i, number 2 i + 1 in the high half.  ``scales`` uint8
[ceil(rows / 128), ceil(K / 128), 32, 4, 4]: the exponent (plus 127) that block b of row r shares is at [r // 128, b // 4, r % 32, r // 32 % 4, b % 4].
A stack of matrices has one more dimension in front of both.

The sizes of weights are those of the repository's own configurations (Llama 3.2 1B, Llama 3.1 8B, experts beside a width of 2,048) and odd ones
beside them; the values of activations are normal with a few channels far larger than the rest, those of weights normal.
"""
from __future__ import annotations

import math

import torch

own = False

#: what the codes 0..15 stand for
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token's activations, rounded to what 4 bits hold: two launches and little else
        {"name": "round-1x2048", "kind": "round", "rows": 1, "k": 2048, "dtype": "bfloat16"},
        # a feed-forward matrix of the 8B shapes out of its float32 checkpoint, quantised as it is loaded and read back
        {"name": "round-14336x4096", "kind": "round", "rows": 14336, "k": 4096, "dtype": "float32"},
        # the embedding rows of a decode step of eight, out of the 1B table in 4 bits
        {"name": "lookup-8", "kind": "lookup", "rows": 128256, "k": 2048, "tokens": 8, "dtype": "float32"},
        # the same for a batch of prompts, an odd number of tokens
        {"name": "lookup-4001", "kind": "lookup", "rows": 128256, "k": 2048, "tokens": 4001, "dtype": "float32"},
        # the smallest contraction of the 1B shapes in a decode step of one
        {"name": "linear-1x2048x2048", "kind": "linear", "m": 1, "n": 2048, "k": 2048, "dtype": "bfloat16"},
        # gate and up of the 8B shapes in a decode step of eight: bound by the weights' bytes
        {"name": "linear-8x28672x4096", "kind": "linear", "m": 8, "n": 28672, "k": 4096, "dtype": "bfloat16"},
        # a batch between decoding and prompts, odd sizes (a last block of scales that is not full), float32 out
        {"name": "linear-77x8191x2080", "kind": "linear", "m": 77, "n": 8191, "k": 2080, "dtype": "float32"},
        # a prompt of 2,048 tokens through a feed-forward matrix of the 8B shapes
        {"name": "linear-2048x14336x4096", "kind": "linear", "m": 2048, "n": 14336, "k": 4096, "dtype": "bfloat16"},
        # both operands in 4 bits, the activations quantised on the way: a short prompt of the 1B shapes, and the prompt of 2,048 tokens
        {"name": "both-200x8192x2048", "kind": "both", "m": 200, "n": 8192, "k": 2048, "dtype": "bfloat16"},
        {"name": "both-2048x14336x4096", "kind": "both", "m": 2048, "n": 14336, "k": 4096, "dtype": "bfloat16"},
        # experts in a decode step of eight tokens with two experts each: most experts get no row or one
        {"name": "experts-16x2048x2048", "kind": "experts", "m": 16, "experts": 32, "n": 2048, "k": 2048, "dtype": "bfloat16"},
        # experts in a prompt of 2,048 tokens with two experts each: runs of very unequal lengths
        {"name": "experts-4096x2048x2048", "kind": "experts", "m": 4096, "experts": 32, "n": 2048, "k": 2048, "dtype": "bfloat16"},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["round", "lookup", "linear", "linear", "both", "experts"])
    dtype = rng.choice(["bfloat16", "float32"])
    k = 32 * _spread(rng, 2, 256)
    if kind == "round":
        return {"kind": kind, "rows": _spread(rng, 1, max(1, 14336 * 4096 // k)), "k": k, "dtype": dtype}
    if kind == "lookup":
        return {"kind": kind, "rows": _spread(rng, 100, 128256 * 2048 // max(k, 2048)), "k": k, "tokens": _spread(rng, 1, 4096 * 2048 // max(k, 2048)), "dtype": dtype}
    if kind == "experts":
        experts = _spread(rng, 2, 64)
        n = _spread(rng, 64, min(8192, 32 * 2048 * 2048 // (experts * k)))
        return {"kind": kind, "m": _spread(rng, 1, 4096), "experts": experts, "n": n, "k": k, "dtype": dtype}
    n = _spread(rng, 64, min(32768, 14336 * 4096 // k))
    return {"kind": kind, "m": _spread(rng, 1, 2048), "n": n, "k": k, "dtype": dtype}


def _tiles(rows, k):
    return -(-rows // 128), -(-k // 128)


def _held(rows, k):
    """Bytes of a matrix in 4 bits: half a byte a number, a byte a block of 32."""
    return rows * k // 2 + rows * k // 32


def work(case):
    k, size = case["k"], 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "round":
        n = case["rows"] * k
        return {"bytes": 2 * size * n, "flops": 2 * n}       # the numbers in, the numbers they are rounded to out
    if case["kind"] == "lookup":
        return {"bytes": _held(case["tokens"], k) + size * case["tokens"] * k + 4 * case["tokens"], "flops": case["tokens"] * k}
    m, n = case["m"], case["n"]
    met = min(m, case.get("experts", 1))                     # at most that many experts' weights have to be read
    return {"bytes": met * _held(n, k) + 2 * m * k + size * m * n, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------ inputs
def _activations(m, k, gen):
    """Normal numbers, one channel in 64 ten times as large: what enters the contractions of a trained decoder."""
    x = torch.randn(m, k, generator=gen, device="cuda")
    loud = torch.rand(k, generator=gen, device="cuda") < 1 / 64
    return x * torch.where(loud, 10.0, 1.0)


def _weights(lead, rows, k, gen):
    """A matrix (or a stack of them) in 4 bits as a loaded model holds it: the numbers of a normal matrix with 1 / K of variance, quantised."""
    scale = k ** -0.5 * torch.exp(0.3 * torch.randn(*lead, rows, 1, generator=gen, device="cuda"))
    data, scales = _quantise(torch.randn(*lead, rows, k, generator=gen, device="cuda") * scale)
    return data, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, k = case["kind"], case["k"]
    state = {"kind": kind, "dtype": DTYPES[case["dtype"]]}
    if kind == "round":
        state["x"] = (_activations(case["rows"], k, gen) if case["rows"] < 1024 else 0.02 * torch.randn(case["rows"], k, generator=gen, device="cuda")).to(state["dtype"])
    elif kind == "lookup":
        state["data"], state["scales"] = _weights((), case["rows"], k, gen)
        state["tokens"] = torch.randint(0, case["rows"], (case["tokens"],), generator=gen, device="cuda", dtype=torch.int32)
    else:
        m = case["m"]
        state["x"] = _activations(m, k, gen).to(torch.bfloat16)
        if kind == "experts":
            experts = case["experts"]
            state["data"], state["scales"] = _weights((experts,), case["n"], k, gen)
            # a router prefers some experts: rows are drawn by weights that differ by a factor of ten and more
            liked = torch.exp(torch.randn(experts, generator=gen, device="cuda"))
            counts = torch.bincount(torch.multinomial(liked, m, replacement=True, generator=gen), minlength=experts)
            state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.cumsum(0)]).to(torch.int32)
            state["longest"] = int(counts.max())
        else:
            state["data"], state["scales"] = _weights((), case["n"], k, gen)
    return state


# ------------------------------------------------------------------------------ plain forms
def _powers(exponents):
    """2 ** (exponents - 127) in float32; 255 stands for no number."""
    e = exponents.to(torch.int32)
    two = (e << 23).view(torch.float32)
    two = torch.where(e == 0, 2.0 ** -127, two)
    return torch.where(e == 255, float("nan"), two)


def _quantise(x):
    """Rows of x in 4 bits.  A block's exponent is the largest with which its largest number stays below 8; the numbers are divided by it and rounded
    to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6, a tie to the one whose last bit is 0, beyond 6 to 6.  A block that holds an infinity or no number
    becomes no number as a whole."""
    lead, rows, k = x.shape[:-2], x.shape[-2], x.shape[-1]
    x = x.float().reshape(*lead, rows, k // 32, 32)
    bits = x.abs().amax(-1).view(torch.int32)                # (the largest of a block with a NaN is NaN, whose exponent is 255 too)
    exponents = ((bits >> 23) - 2).clamp_min(0)
    no = (bits >> 23) == 255
    # 2 ** (127 - exponent): 254 - exponent lies between 2 and 254
    y = x.abs() * ((254 - exponents) << 23).view(torch.float32)[..., None]
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)).to(torch.uint8)
    code = torch.where(no[..., None], 0, code | (torch.signbit(x).to(torch.uint8) << 3)).to(torch.uint8)
    code = code.reshape(*lead, rows, k // 2, 2)
    data = code[..., 0] | (code[..., 1] << 4)
    exponents = torch.where(no, 255, exponents).to(torch.uint8)
    tr, tk = _tiles(rows, k)
    full = torch.zeros(*lead, tr * 128, tk * 4, dtype=torch.uint8, device=x.device)
    full[..., :rows, : k // 32] = exponents
    n = len(lead)
    full = full.reshape(*lead, tr, 4, 32, tk, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    return data, full.contiguous()


def _numbers(data, scales):
    """What a matrix (or a stack) in 4 bits stands for, in float32."""
    lead, rows, k = data.shape[:-2], data.shape[-2], 2 * data.shape[-1]
    code = torch.stack([data & 15, data >> 4], -1).reshape(*lead, rows, k // 32, 32)
    values = torch.tensor(VALUES, device=data.device)[code.to(torch.int32)]
    n = len(lead)
    tr, tk = scales.shape[n], scales.shape[n + 1]
    e = scales.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).reshape(*lead, tr * 128, tk * 4)[..., :rows, : k // 32]
    return (values * _powers(e)[..., None]).reshape(*lead, rows, k)


def _plain(state):
    kind, dtype = state["kind"], state["dtype"]
    if kind == "round":
        return _numbers(*_quantise(state["x"])).to(dtype)
    if kind == "lookup":
        tokens = state["tokens"].long()
        tk = state["scales"].shape[1]
        code = state["data"][tokens]
        values = torch.tensor(VALUES, device=code.device)[torch.stack([code & 15, code >> 4], -1).to(torch.int32)].reshape(len(tokens), -1, 32)
        e = state["scales"][tokens // 128, :, tokens % 32, tokens // 32 % 4].reshape(len(tokens), tk * 4)[:, : values.shape[1]]
        return (values * _powers(e)[..., None]).reshape(len(tokens), -1).to(dtype)
    w = _numbers(state["data"], state["scales"])
    if kind == "linear":
        return (state["x"].float() @ w.t()).to(dtype)
    if kind == "both":
        return (_numbers(*_quantise(state["x"])) @ w.t()).to(dtype)
    # experts: every run padded to the longest one
    x, offsets = state["x"].float(), state["offsets"].long()
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    place = row - offsets[expert]
    padded = x.new_zeros(w.shape[0], state["longest"], x.shape[1])
    padded[expert, place] = x
    return torch.bmm(padded, w.transpose(1, 2))[expert, place].to(dtype)


def run(state):
    if not own:
        return _plain(state)
    from fastgguf_b200 import ops
    kind, dtype = state["kind"], state["dtype"]
    if kind == "round":
        return ops.mxfp4_rows(ops.mxfp4_quantize(state["x"]), out_dtype=dtype)
    w = ops.Mxfp4(state["data"], state["scales"])
    if kind == "lookup":
        return ops.mxfp4_rows(w, state["tokens"], out_dtype=dtype)
    if kind == "linear":
        return ops.gemm_mxfp4(state["x"], w, out_dtype=dtype)
    if kind == "both":
        return ops.gemm_mxfp4_both(ops.mxfp4_quantize(state["x"]), w, out_dtype=dtype)
    return ops.gemm_mxfp4_grouped(state["x"], w, state["offsets"], out_dtype=dtype)


# ------------------------------------------------------------------------------ the definition in 64 bits
def _exact_numbers(data, scales, rows=None):
    """Number by number: the sign, the two exponent bits and the mantissa bit of a code, times its block's power of two."""
    rows = torch.arange(data.shape[0], device=data.device) if rows is None else rows
    byte = data[rows].long()
    code = torch.empty(len(rows), 2 * data.shape[1], dtype=torch.int64, device=data.device)
    code[:, 0::2], code[:, 1::2] = byte % 16, byte // 16
    exponent, mantissa = code // 2 % 4, (code % 2).double()
    size = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2.0 ** (exponent - 1).double())
    block = torch.arange(code.shape[1], device=data.device) // 32
    r = rows[:, None]
    shared = scales[r // 128, block // 4, r % 32, r // 32 % 4, block % 4].long()
    value = torch.where(code >= 8, -size, size) * _two(shared - 127)
    return torch.where(shared == 255, float("nan"), value)


def _two(n):
    return ((n.long() + 1023) << 52).view(torch.float64)


def _exact_rounded(x):
    x = x.double().reshape(x.shape[0], -1, 32)
    largest = x.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(largest)                              # largest = m 2^e with 1/2 <= m < 1
    e = torch.where(largest == 0, -127, (e - 3).clamp_min(-127))
    y = x * _two(-e)
    _, f = torch.frexp(y)
    step = _two((f - 1).clamp_min(0) - 1)                    # the distance of neighbours: 1/2 below 2, 1 below 4, 2 from there
    y = (torch.round(y / step) * step).clamp(-6, 6)
    value = y * _two(e)
    return torch.where(torch.isfinite(largest), value, float("nan")).reshape(x.shape[0], -1)


def exact(case, seed):
    state = prepare(case, seed)
    kind = state["kind"]
    if kind == "round":
        return _exact_rounded(state["x"])
    if kind == "lookup":
        return _exact_numbers(state["data"], state["scales"], state["tokens"].long())
    if kind == "experts":
        x, bounds = state["x"].double(), state["offsets"].tolist()
        parts = [x[a:b] @ _exact_numbers(state["data"][e], state["scales"][e]).t() for e, (a, b) in enumerate(zip(bounds, bounds[1:])) if b > a]
        return torch.cat(parts)
    x = state["x"].double() if kind == "linear" else _exact_rounded(state["x"])
    return x @ _exact_numbers(state["data"], state["scales"]).t()
