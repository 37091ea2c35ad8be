"""Matrices in microscaled 4-bit floating point at the edges of what their calls allow."""
import pytest
import torch

import plain_mxfp4 as plain
from fastgguf_b200 import ops
from fastgguf_b200.ops import Mxfp4


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(m, k, seed):
    return torch.randn(m, k, generator=_gen(seed)).bfloat16()


# ------------------------------------------------------------------------------ padding exponents
def _padded(data, e, byte):
    """The matrix (or stack) with every exponent of a row or block past it set to `byte`."""
    padding = Mxfp4.from_exponents(data, torch.ones_like(e)).scales == 0
    w = Mxfp4.from_exponents(data, e)
    return Mxfp4(data.contiguous().cuda(), torch.where(padding, torch.tensor(byte, dtype=torch.uint8), w.scales).cuda())


def test_padding_is_every_place_past_the_matrix():
    data, e = plain.random_matrix(130, 160, _gen(1))
    full = Mxfp4.from_exponents(data, torch.ones_like(e)).scales
    assert full.shape == (2, 2, 32, 4, 4) and int((full == 0).sum()) == full.numel() - 130 * 5


@pytest.mark.gpu
@pytest.mark.parametrize("k", [32, 96, 160, 352, 448])
@pytest.mark.parametrize("m", [1, 8, 12, 200])
def test_padding_exponents_change_no_bit(m, k):
    """Any byte but 255 may stand behind the rows and blocks of a matrix, of the weights' and of quantised activations' alike."""
    n, X = 140, 3
    data, e = plain.random_matrix(n, k, _gen(n + k))
    many, many_e = data.expand(X, n, k // 2).clone(), e.expand(X, n, k // 32).clone()
    many[1], many_e[1] = plain.random_matrix(n, k, _gen(k))
    rows_data, rows_e = plain.random_matrix(m, k, _gen(m + k))
    x = _rows(m, k, m).cuda()
    odd = torch.zeros(m, k + 1, dtype=torch.bfloat16, device="cuda")              # rows that TMA cannot address
    odd[:, :k] = x
    cut = torch.tensor([0, m // 2, m // 2, m], dtype=torch.int32, device="cuda")

    def results(byte):
        w, stack, q = _padded(data, e, byte), _padded(many, many_e, byte), _padded(rows_data, rows_e, byte)
        return [ops.gemm_mxfp4(x, w), ops.gemm_mxfp4(odd[:, :k], w), ops.gemm_mxfp4(x, w, out_dtype=torch.float32), ops.gemm_mxfp4_both(q, w, out_dtype=torch.float32),
                ops.gemm_mxfp4_grouped(x, stack, cut), ops.gemm_mxfp4_grouped(odd[:, :k], stack, cut), ops.mxfp4_rows(w)]

    want = results(0)
    assert all(torch.isfinite(t).all() for t in want)
    for byte in (126, 252, 253, 254):
        for i, (got, zero) in enumerate(zip(results(byte), want)):
            assert torch.equal(got, zero), (byte, i)


# ------------------------------------------------------------------------------ outputs as the weights of the next kernel
def test_only_the_quantiser_releases_its_successor_early():
    """What the other kernels write may be weights, which a bfloat16 or float32 contraction fetches before it waits for the kernels in front of it."""
    import os
    import re
    from fastgguf_b200.csrc import build
    releasing = set()
    for name in ("mxfp4.cu", "mxfp4.cuh", "mxfp4_tc.cuh", "gemm_mxfp4.cu", "gemm_mxfp4_both.cuh"):
        with open(os.path.join(build.CSRC_DIR, name)) as f:
            code = re.sub(r"//[^\n]*", "", f.read())
        for part in code.split("__global__")[1:]:
            if "pdl_launch_dependents" in part or "griddepcontrol.launch_dependents" in part:
                releasing.add(re.search(r"(\w+_kernel)\(", part).group(1))
    assert releasing == {"mxfp4_quantize_kernel"}


def _random(n, k, seed, lead=()):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*lead, n, k, generator=g, device="cuda") * k ** -0.5).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("n", [8, 48, 640, 2048])
def test_an_output_is_the_weight_of_the_next_contraction(n, rows):
    """The contractions write W, the next kernel of the stream (or the one behind that) reads it as its weights: as if the device were waited for in between."""
    from fastgguf_b200.ops import fast_gemm
    k, mid = 1024, 512
    w = ops.mxfp4_quantize(_random(mid, k, 1))
    stack = ops.mxfp4_quantize(_random(mid, k, 2, (2,)))
    cut = torch.tensor([0, n // 3, n], dtype=torch.int32, device="cuda")
    inputs = [_random(n, k, 10 + i) for i in range(6)]
    packed = [ops.mxfp4_quantize(t) for t in inputs]
    a, a32 = _random(rows, mid, 3), _random(rows, mid, 4).float()
    other = _random(256, mid, 5)
    made, made32 = torch.zeros(n, mid, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, mid, device="cuda")
    writers = [lambda i, out: ops.gemm_mxfp4(inputs[i], w, out=out), lambda i, out: ops.gemm_mxfp4_both(packed[i], w, out=out),
               lambda i, out: ops.gemm_mxfp4_grouped(inputs[i], stack, cut, out=out)]
    f32 = fast_gemm.gemm_f32_stream if rows <= 16 else fast_gemm.gemm_f32

    def chain(write, i, wait):
        write(i, made)
        if wait:
            torch.cuda.synchronize()
        got = [fast_gemm.gemm_tc(a, made)]
        write((i + 1) % len(inputs), made)
        if wait:
            torch.cuda.synchronize()
        fast_gemm.gemm_tc(a, other)                          # (a kernel between that releases its successor before it waits)
        got.append(fast_gemm.gemm_tc(a, made))
        write(i, made32)
        if wait:
            torch.cuda.synchronize()
        got.append(f32(a32, made32))
        return got

    for write in writers:
        want = [[t.clone() if t is not None else None for t in chain(write, i, True)] for i in range(len(inputs))]
        assert want[0][0] is not None and not torch.equal(want[0][0], want[1][0])
        got = [chain(write, i, False) for _ in range(10) for i in range(len(inputs))]
        torch.cuda.synchronize()
        for j, g in enumerate(got):
            for x, y in zip(g, want[j % len(inputs)]):
                assert (x is None and y is None) or torch.equal(x, y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            recorded = [chain(write, i, False) for i in range(len(inputs))]
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        for g, y in zip(recorded, want):
            assert all((p is None and q is None) or torch.equal(p, q) for p, q in zip(g, y))
    ops.raise_on_device_error("chains")


# ------------------------------------------------------------------------------ long rows
def test_launchers_refuse_rows_whose_end_passes_31_bits():
    """Before they touch the device or the memory (the addresses here are none)."""
    from ctypes import c_void_p
    L, refused, at = ops.lib("mx"), 10002, c_void_p(1 << 20)                      # (FG_ERR_BAD_SIZE)
    for k in (2 ** 31 - 32, 2 ** 31 - 128, 2 ** 31 - 480):
        assert L.fg_gemm_mxfp4(at, k, at, at, at, 1, 4, 0, 1, 4, k, None) == refused
        assert L.fg_gemm_mxfp4_both(at, at, at, at, at, 1, 4, 0, 1, 4, k, None) == refused
        assert L.fg_gemm_mxfp4_grouped(at, k, at, at, at, 2, at, 1, 4, 0, 1, 4, k, None) == refused
        assert L.fg_mxfp4_quantize(at, 0, k, 0, at, at, 1, 1, k, None) == refused
        assert L.fg_mxfp4_rows(at, at, at, at, 0, k, 1, 1, k, 1.0, None) == refused


@pytest.mark.gpu
@pytest.mark.parametrize("k", [2 ** 29 + 160, 3 * 2 ** 28 + 96])
def test_the_end_of_a_long_row(k):
    """Rows whose exponents take more than 2^31 bytes: numbers behind that place count as they should."""
    n = 3
    data, scales = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda"), torch.zeros(1, (k + 127) // 128, 32, 4, 4, dtype=torch.uint8, device="cuda")
    tail_data, tail_e = plain.random_matrix(n, 320, _gen(1))
    first = (k - 320) // 32                                    # the block where the last 320 numbers start
    data[:, -160:] = tail_data.cuda()
    for r in range(n):
        for b in range(10):
            scales[0, (first + b) // 4, r, 0, (first + b) % 4] = tail_e[r, b]
    w = Mxfp4(data, scales)
    x = torch.zeros(1, k, dtype=torch.bfloat16, device="cuda")
    x[:, -320:] = _rows(1, 320, 2).cuda()
    x[:, 64:96] = 1.0                                          # (under weights of zero)
    want, slack = plain.product(x[:, -320:].cpu(), plain.numbers(tail_data, tail_e))
    plain.check(ops.gemm_mxfp4(x, w, out_dtype=torch.float32), want, slack)
    q = ops.mxfp4_quantize(x)
    rounded = plain.rounded(x[:, -320:].cpu())[0]
    assert torch.equal(ops.mxfp4_rows(q, out_dtype=torch.bfloat16)[:, -320:].double().cpu(), rounded)
    want, slack = plain.product(rounded, plain.numbers(tail_data, tail_e))
    plain.check(ops.gemm_mxfp4_both(q, w, out_dtype=torch.float32), want, slack)


# ------------------------------------------------------------------------------ sizes beyond 31 bits
def test_sizes_beyond_31_bits_are_refused_not_cut(monkeypatch):
    from fastgguf_b200.ops import KernelError, mxfp4
    monkeypatch.setattr(mxfp4, "require_cuda", lambda *t: None)
    monkeypatch.setattr(mxfp4, "_on_one_device", lambda *t: 0)
    monkeypatch.setattr(mxfp4, "_launch", lambda *a: pytest.fail("a refused call reached a kernel"))

    def tensor(*shape, dtype=torch.uint8):
        return torch.empty(*shape, dtype=dtype, device="meta")

    def matrix(rows, k, lead=()):
        return Mxfp4(tensor(*lead, rows, k // 2), tensor(*lead, (rows + 127) // 128, (k + 127) // 128, 32, 4, 4))

    many = 2 ** 32 + 32                                    # would reach a kernel as 32
    small = matrix(4, 64)
    calls = [
        lambda: ops.mxfp4_quantize(tensor(many, 64, dtype=torch.float32)),
        lambda: ops.mxfp4_quantize(tensor(2, many, dtype=torch.bfloat16)),
        lambda: ops.mxfp4_quantize(tensor(many, 2, 64, dtype=torch.bfloat16)),
        lambda: ops.mxfp4_rows(matrix(many, 64)),
        lambda: ops.mxfp4_rows(matrix(4, many)),
        lambda: ops.mxfp4_rows(small, tensor(many, dtype=torch.int32)),
        lambda: ops.gemm_mxfp4(tensor(many, 64, dtype=torch.bfloat16), small),
        lambda: ops.gemm_mxfp4(tensor(2, 64, dtype=torch.bfloat16), matrix(many, 64)),
        lambda: ops.gemm_mxfp4(tensor(2, many, dtype=torch.bfloat16), matrix(4, many)),
        lambda: ops.gemm_mxfp4_both(matrix(many, 64), small),
        lambda: ops.gemm_mxfp4_both(matrix(2, many), matrix(4, many)),
        lambda: ops.gemm_mxfp4_grouped(tensor(many, 64, dtype=torch.bfloat16), matrix(4, 64, (3,)), tensor(4, dtype=torch.int32)),
    ]
    for call in calls:
        with pytest.raises(KernelError, match="sizes go up to"):
            call()


# ------------------------------------------------------------------------------ many rows
@pytest.mark.gpu
@pytest.mark.parametrize("stride", [33, 0])
@pytest.mark.parametrize("m", [65535 * 16, 65535 * 16 + 1, 2 * 65535 * 16 + 37])
def test_more_rows_than_a_grid_takes_where_tma_cannot_address_them(m, stride):
    n, k = 5, 32
    data, e = plain.random_matrix(n, k, _gen(1))
    w, numbers = Mxfp4.from_exponents(data.cuda(), e.cuda()), plain.numbers(data, e)
    if stride:
        x = torch.randn(m, stride, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").bfloat16()[:, :k]
    else:
        x = _rows(1, k, 3).cuda().expand(m, k)
    want, slack = plain.product(x.cpu(), numbers)
    for dtype in (torch.bfloat16, torch.float32):
        room = torch.full((m + 2, n + 1), 7.0, dtype=dtype, device="cuda")
        ops.gemm_mxfp4(x, w, out=room[1:m + 1, :n])
        plain.check(room[1:m + 1, :n], want, slack)
        room[1:m + 1, :n] = 7.0
        assert (room == 7.0).all()
    total = torch.ones(m, n, device="cuda")
    ops.gemm_mxfp4(x, w, out=total, accumulate=True)
    plain.check(total, want + 1.0, slack + 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead,rows,k", [((65536,), 1, 32), ((33000,), 129, 160), ((), 65535 * 128 + 1, 32), ((), 65537 * 128, 64)])
def test_quantising_more_tiles_than_a_grids_second_dimension(dtype, lead, rows, k):
    x = torch.randn(*lead, rows, k, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    q = ops.mxfp4_quantize(x)
    if lead:
        for i in (0, 1, 32767, lead[0] - 1):
            want, e = plain.rounded(x[i])
            assert torch.equal(q[i].exponents().cpu(), e) and torch.equal(plain.of(q[i]), want)
        some = torch.randint(0, lead[0], (200,), generator=_gen(2)).tolist()
        data, e = zip(*((q[i].data, q[i].exponents()) for i in some))
        want, want_e = plain.rounded(x[some].reshape(-1, k))
        assert torch.equal(torch.cat(e).cpu(), want_e) and torch.equal(plain.numbers(torch.cat(data), torch.cat(e)), want)
    else:
        back = ops.mxfp4_rows(q)
        for at in (0, 127, 4194304, rows - 300):
            assert torch.equal(back[at:at + 300].double().cpu(), plain.rounded(x[at:at + 300])[0])


def test_named_kernels_refuse_what_the_header_does_not_allow():
    """Before they touch the device or the memory (the addresses here are none)."""
    from ctypes import c_void_p
    L, refused, at = ops.lib("mx"), 10002, c_void_p(1 << 20)                      # (FG_ERR_BAD_SIZE)
    for form, bn, splits in [(2, 0, 1), (2, 24, 1), (2, 272, 1), (2, 64, 0), (2, 64, 9), (3, 48, 1), (3, 64, 2), (3, 64, 0), (4, 64, 1), (-1, 64, 1)]:
        assert L.fg_gemm_mxfp4_ext(at, 64, at, at, at, 1, 64, 0, 100, 64, 64, form, bn, splits, None) == refused, (form, bn, splits)
    for bn, splits in [(128, 0), (128, 9), (112, 0), (96, 1), (24, 1), (272, 1)]:  # (96: does not take 100 rows)
        assert L.fg_gemm_mxfp4_both_ext(at, at, at, at, at, 1, 64, 0, 100, 64, 64, bn, splits, None) == refused, (bn, splits)


def test_blocks_that_keep_their_halves_apart_are_reordered_as_the_text_says():
    """Byte j of a block: number j below, number j + 16 above."""
    numbers = torch.randint(0, 16, (3, 5, 32), generator=_gen(1), dtype=torch.uint8)         # codes [rows, blocks, 32]
    raw = numbers[..., :16] | numbers[..., 16:] << 4
    codes = torch.cat([raw & 15, raw >> 4], -1)
    data = (codes[..., 0::2] | codes[..., 1::2] << 4).flatten(-2)
    e = torch.randint(100, 140, (3, 5), generator=_gen(2), dtype=torch.uint8)
    w = Mxfp4.from_exponents(data, e)
    want = plain.VALUES[numbers.long()] * torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double() - 127)[..., None]
    assert torch.equal(plain.of(w), want.reshape(3, 160))
