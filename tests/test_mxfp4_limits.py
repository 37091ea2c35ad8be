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
