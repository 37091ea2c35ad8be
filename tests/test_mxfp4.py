"""Matrices in microscaled 4-bit floating point: the layout and the refusals (CPU), the kernels against plain float64 (GPU)."""
import pytest
import torch

import plain_mxfp4 as plain
from fastgguf_b200 import ops
from fastgguf_b200.ops import KernelError, Mxfp4


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _matrix(rows, k, seed, **kw):
    data, e = plain.random_matrix(rows, k, _gen(seed), **kw)
    return Mxfp4.from_exponents(data.cuda(), e.cuda()), plain.numbers(data, e)


def _rows(m, k, seed, loud=True):
    g = _gen(seed)
    x = torch.randn(m, k, generator=g)
    if loud:
        x = x * torch.where(torch.rand(k, generator=g) < 1 / 64, 20.0, 1.0)
    return x.bfloat16()


# ------------------------------------------------------------------------------ layout and refusals, no device
@pytest.mark.parametrize("lead", [(), (3,)])
@pytest.mark.parametrize("rows,k", [(1, 32), (128, 128), (129, 160), (300, 96)])
def test_exponents_stand_where_the_layout_says(lead, rows, k):
    g = _gen(rows + k)
    data = torch.randint(0, 256, (*lead, rows, k // 2), generator=g, dtype=torch.uint8)
    e = torch.randint(0, 255, (*lead, rows, k // 32), generator=g, dtype=torch.uint8)
    w = Mxfp4.from_exponents(data, e)
    assert w.shape == (*lead, rows, k) and torch.equal(w.exponents(), e)
    scales, flat = (w.scales[2], e[2]) if lead else (w.scales, e)
    for r in (0, rows // 2, rows - 1):
        for b in range(k // 32):
            assert scales[r // 128, b // 4, r % 32, r // 32 % 4, b % 4] == flat[r, b]
    if lead:
        assert torch.equal(w[1].exponents(), e[1]) and torch.equal(w[1].data, data[1])


def test_containers_of_other_shapes_are_refused():
    data, e = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    w = Mxfp4.from_exponents(data, e)
    with pytest.raises(KernelError, match="uint8"):
        Mxfp4(data.to(torch.int16), w.scales)
    with pytest.raises(KernelError, match="whole blocks"):
        Mxfp4(torch.zeros(4, 20, dtype=torch.uint8), w.scales)
    with pytest.raises(KernelError, match="whole blocks"):
        Mxfp4(torch.zeros(4, 0, dtype=torch.uint8), w.scales)
    with pytest.raises(KernelError, match="scales of"):
        Mxfp4(torch.zeros(129, 32, dtype=torch.uint8), w.scales)
    with pytest.raises(KernelError, match="contiguous"):
        Mxfp4(torch.zeros(4, 64, dtype=torch.uint8)[:, ::2], w.scales)
    with pytest.raises(KernelError, match="X, rows"):
        Mxfp4(torch.zeros(32, dtype=torch.uint8), w.scales)
    with pytest.raises(KernelError, match="exponents"):
        Mxfp4.from_exponents(data, torch.zeros(4, 3, dtype=torch.uint8))
    with pytest.raises(KernelError, match="stack"):
        w[0]


def test_there_is_no_cpu_path():
    w = Mxfp4.from_exponents(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.mxfp4_quantize(x), lambda: ops.mxfp4_rows(w), lambda: ops.gemm_mxfp4(x, w), lambda: ops.gemm_mxfp4_both(w, w),
                 lambda: ops.gemm_mxfp4_grouped(x, w, torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(KernelError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_tensors_on_two_devices_are_refused():
    w, _ = _matrix(4, 64, 1)
    here = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.gemm_mxfp4(here, w), lambda: ops.gemm_mxfp4(here.cuda(), w, out=torch.zeros(2, 4)), lambda: ops.mxfp4_rows(w, torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(KernelError, match="cpu"):
            call()


@pytest.fixture
def no_device_check(monkeypatch):
    from fastgguf_b200.ops import mxfp4
    monkeypatch.setattr(mxfp4, "require_cuda", lambda *t: None)
    monkeypatch.setattr(mxfp4, "_on_one_device", lambda *t: 0)
    monkeypatch.setattr(mxfp4, "_launch", lambda *a: pytest.fail("a refused call reached a kernel"))


def test_calls_that_do_not_fit_are_refused_before_a_launch(no_device_check):
    w = Mxfp4.from_exponents(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))
    other = Mxfp4.from_exponents(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))
    stack = Mxfp4.from_exponents(torch.zeros(3, 4, 32, dtype=torch.uint8), torch.zeros(3, 4, 2, dtype=torch.uint8))
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    offsets = torch.zeros(4, dtype=torch.int32)
    wide = torch.zeros(2, 128, dtype=torch.bfloat16)
    refusals = [
        ("float32 or bfloat16", lambda: ops.mxfp4_quantize(x.half())),
        ("whole blocks", lambda: ops.mxfp4_quantize(x[:, :40])),
        ("contiguous", lambda: ops.mxfp4_quantize(wide[:, ::2])),
        ("rows, K", lambda: ops.mxfp4_quantize(x[0])),
        ("not a stack", lambda: ops.mxfp4_rows(stack)),
        ("int32", lambda: ops.mxfp4_rows(w, torch.zeros(2, dtype=torch.int64))),
        ("int32", lambda: ops.mxfp4_rows(w, torch.zeros(2, 2, dtype=torch.int32))),
        ("cannot write", lambda: ops.mxfp4_rows(w, out_dtype=torch.float16)),
        ("out must be", lambda: ops.mxfp4_rows(w, out=torch.zeros(3, 64))),
        ("out must be", lambda: ops.mxfp4_rows(w, out=torch.zeros(64, 4).t())),
        ("bfloat16", lambda: ops.gemm_mxfp4(x.float(), w)),
        ("activations are", lambda: ops.gemm_mxfp4(wide, w)),
        ("contiguous", lambda: ops.gemm_mxfp4(wide[:, ::2], w)),
        ("not a stack", lambda: ops.gemm_mxfp4(x, stack)),
        ("out must be", lambda: ops.gemm_mxfp4(x, w, out=torch.zeros(2, 5))),
        ("out must be", lambda: ops.gemm_mxfp4(x, w, out=torch.zeros(1, 4).expand(2, 4))),
        ("out must be", lambda: ops.gemm_mxfp4(x, w, out=torch.zeros(2, 4), out_dtype=torch.bfloat16)),
        ("cannot write", lambda: ops.gemm_mxfp4(x, w, out_dtype=torch.float16)),
        ("accumulate needs the tensor", lambda: ops.gemm_mxfp4(x, w, accumulate=True)),
        ("32-bit", lambda: ops.gemm_mxfp4(x, w, out=torch.zeros(2, 4, dtype=torch.bfloat16), accumulate=True)),
        ("but w is", lambda: ops.gemm_mxfp4_both(other, w)),
        ("one matrix each", lambda: ops.gemm_mxfp4_both(stack, w)),
        ("stack of matrices", lambda: ops.gemm_mxfp4_grouped(x, w, offsets)),
        ("offsets", lambda: ops.gemm_mxfp4_grouped(x, stack, offsets[:3])),
        ("offsets", lambda: ops.gemm_mxfp4_grouped(x, stack, offsets.long())),
    ]
    for match, call in refusals:
        with pytest.raises(KernelError, match=match):
            call()


def test_launchers_refuse_rows_beyond_31_bits_and_other_widths(no_device_check):
    """Before they touch the device or the memory (the addresses here are none)."""
    from ctypes import c_void_p
    L, refused, most, at = ops.lib("mx"), 10002, 2 ** 31 - 1, c_void_p(1 << 20)          # (FG_ERR_BAD_SIZE)
    sizes = [(most, 64), (most - 500, 64), (4, most), (4, most - 500)]
    for M, N in sizes:
        assert L.fg_gemm_mxfp4(at, 32, at, at, at, 1, N, 0, M, N, 32, None) == refused
        for form in (1, 2, 3):
            assert L.fg_gemm_mxfp4_ext(at, 32, at, at, at, 1, N, 0, M, N, 32, form, 16, 1, None) == refused
            assert L.fg_gemm_mxfp4_ext(at, 32, at, at, at, 1, N, 0, M, N, 32, form, 32, 1, None) == refused
        assert L.fg_gemm_mxfp4_both(at, at, at, at, at, 1, N, 0, M, N, 32, None) == refused
        assert L.fg_gemm_mxfp4_grouped(at, 32, at, at, at, 2, at, 1, N, 0, M, N, 32, None) == refused
    for bn in (0, 8, 16, 48, 240, 272):                                                       # a pair's tiles are multiples of 32 tokens
        assert L.fg_gemm_mxfp4_ext(at, 32, at, at, at, 1, 64, 0, 64, 64, 32, 3, bn, 1, None) == refused
    assert L.fg_gemm_mxfp4_grouped(at, 32, at, at, at, 1000, at, 1, 3000000, 0, 4, 3000000, 32, None) == refused       # 3 10^9 rows of all experts


# ------------------------------------------------------------------------------ quantising and reading rows
def _border_rows():
    """Rows whose blocks hold the borders between codes and their neighbours, under maxima that set the exponent."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.5, 1.0, 2.0, 4.0])
    near = torch.cat([mids, torch.nextafter(mids, torch.tensor(0.0)), torch.nextafter(mids, torch.tensor(9.0))])[:30]
    rows = []
    for top in (4.0, 7.9999995, 6.0, 5.0, 7.0):
        for sign in (1.0, -1.0):
            rows.append(torch.cat([torch.tensor([sign * top, 0.0]), sign * near.clamp_max(top)]))
    x = torch.stack(rows)
    return torch.cat([x * 2.0 ** p for p in (-126, -100, -20, 0, 3, 60, 123)])


@pytest.mark.gpu
def test_quantiser_at_the_borders_between_codes():
    x = _border_rows()
    want, e = plain.rounded(x)
    q = ops.mxfp4_quantize(x.cuda())
    assert torch.equal(q.exponents().cpu(), e)
    assert torch.equal(plain.of(q), want)
    b = x.bfloat16()
    want, e = plain.rounded(b)
    q = ops.mxfp4_quantize(b.cuda())
    assert torch.equal(q.exponents().cpu(), e) and torch.equal(plain.of(q), want)


@pytest.mark.gpu
def test_quantiser_of_small_large_and_no_numbers():
    tiny = 2.0 ** -149
    rows = [torch.zeros(32), torch.full((32,), tiny), torch.full((32,), 2.0 ** -127), torch.full((32,), 1.5 * 2.0 ** -126), torch.full((32,), 3.4028234e38),
            torch.cat([torch.tensor([float("inf")]), torch.ones(31)]), torch.cat([torch.ones(31), torch.tensor([float("nan")])]),
            torch.cat([torch.tensor([-float("inf"), float("nan")]), torch.zeros(30)]), -torch.linspace(0, 1, 32), torch.full((32,), -0.0)]
    x = torch.stack(rows)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        want, e = plain.rounded(y)
        q = ops.mxfp4_quantize(y.cuda())
        assert torch.equal(q.exponents().cpu(), e)
        assert torch.equal(torch.nan_to_num(plain.of(q), nan=7e77), torch.nan_to_num(want, nan=7e77))
        back = ops.mxfp4_rows(q)
        assert torch.equal(torch.nan_to_num(back.cpu(), nan=7e30), torch.nan_to_num(want.float(), nan=7e30))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 2048), (3, 96), (31, 160), (127, 128), (128, 4096), (129, 352), (1000, 2080)])
def test_quantiser_over_sizes_and_strides(dtype, rows, k):
    g = _gen(rows * 7 + k)
    wide = (torch.randn(rows, k + 8, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(dtype)
    for x in (wide[:, :k].contiguous(), wide[:, 8:], wide[:, 3:k + 3]):        # aligned, with a stride, and off the 16-byte grid
        want, e = plain.rounded(x)
        dev = wide.cuda()
        off = x.storage_offset() if not x.is_contiguous() else 0
        y = x.cuda() if x.is_contiguous() else dev[:, off:off + k]
        q = ops.mxfp4_quantize(y)
        assert torch.equal(q.exponents().cpu(), e) and torch.equal(plain.of(q), want)
        tr, tk = q.scales.shape[:2]
        assert int((q.scales == 255).sum()) == 0 and (tr, tk) == ((rows + 127) // 128, (k + 127) // 128)


@pytest.mark.gpu
def test_quantiser_of_a_stack():
    x = torch.randn(3, 130, 96, generator=_gen(5)).bfloat16()
    q = ops.mxfp4_quantize(x.cuda())
    for i in range(3):
        want, e = plain.rounded(x[i])
        assert torch.equal(q[i].exponents().cpu(), e) and torch.equal(plain.of(q[i]), want)
    every_other = torch.randn(6, 40, 64, generator=_gen(6)).cuda()
    q = ops.mxfp4_quantize(every_other[::2])
    assert torch.equal(plain.of(q[1]), plain.rounded(every_other[2])[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_code_under_every_exponent(dtype):
    data = torch.arange(16, dtype=torch.uint8).repeat(256, 1) * 17           # sixteen bytes: each code twice
    e = torch.arange(256, dtype=torch.uint8)[:, None]
    w = Mxfp4.from_exponents(data.cuda(), e.cuda())
    got = ops.mxfp4_rows(w, out_dtype=dtype).cpu()
    want = plain.numbers(data, e).to(torch.float32).to(dtype)                 # (beyond float32's range: infinity)
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))
    assert torch.isnan(got[255]).all() and not torch.isnan(got[:255]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k,n", [(5, 32, 1), (300, 96, 7), (1000, 2048, 130), (77, 2080, 4001)])
def test_lookup(dtype, rows, k, n):
    w, numbers = _matrix(rows, k, rows + k)
    index = torch.randint(0, rows, (n,), generator=_gen(n), dtype=torch.int32)
    index[0] = rows - 1
    index[n // 2] = 0
    want = numbers[index.long()]
    got = ops.mxfp4_rows(w, index.cuda(), out_dtype=dtype)
    assert torch.equal(got.cpu().double(), want)                             # a number of the format is exact in either type
    scaled = ops.mxfp4_rows(w, index.cuda(), scale=45.254834, out_dtype=dtype)
    factor = torch.tensor(45.254834, dtype=torch.float32).double()
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    assert ((scaled.cpu().double() - want * factor).abs() <= (half + 1.01 * 2.0 ** -24) * (want * factor).abs()).all()
    wide = torch.full((n, k + 3), 7.0, dtype=dtype, device="cuda")
    ops.mxfp4_rows(w, index.cuda(), out=wide[:, 1:k + 1])
    assert torch.equal(wide[:, 1:k + 1].cpu().double(), want) and (wide[:, 0] == 7).all() and (wide[:, k + 1:] == 7).all()


@pytest.mark.gpu
def test_lookup_of_rows_that_are_not_there_and_of_none():
    w, numbers = _matrix(10, 64, 3)
    got = ops.mxfp4_rows(w, torch.tensor([3, -1, 10, 9, 2 ** 31 - 1], dtype=torch.int32, device="cuda")).cpu()
    assert torch.isnan(got[[1, 2, 4]]).all() and torch.equal(got[[0, 3]].double(), numbers[[3, 9]])
    assert ops.mxfp4_rows(w, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 64)
    assert ops.mxfp4_quantize(torch.zeros(0, 64, device="cuda")).shape == (0, 64)


# ------------------------------------------------------------------------------ contractions
SIZES = [(1, 64, 32), (1, 2048, 2048), (2, 1, 64), (3, 65, 96), (8, 128, 128), (9, 200, 160), (15, 300, 1056), (16, 256, 4096), (17, 129, 224),
         (33, 500, 512), (64, 384, 2048), (65, 127, 640), (100, 1000, 352), (129, 257, 2080), (256, 256, 1024), (300, 640, 96), (513, 320, 800)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SIZES)
def test_contraction(m, n, k):
    x, (w, numbers) = _rows(m, k, m + n), _matrix(n, k, n + k)
    want, slack = plain.product(x, numbers)
    xd = x.cuda()
    plain.check(ops.gemm_mxfp4(xd, w), want, slack)
    got = ops.gemm_mxfp4(xd, w, out_dtype=torch.float32)
    plain.check(got, want, slack)
    assert torch.equal(got, ops.gemm_mxfp4(xd, w, out_dtype=torch.float32))              # the order of sums is fixed
    res = torch.randn(m, n, generator=_gen(1)).cuda()
    out = res.clone()
    assert ops.gemm_mxfp4(xd, w, out=out, accumulate=True) is out
    plain.check(out, want + res.double().cpu(), slack + 2.0 ** -24 * res.double().cpu().abs())


def _named(x, w, form, bn=16, splits=1, dtype=torch.float32):
    """The contraction by a kernel of the test's choice, into rows with a stride."""
    m, n = x.shape[0], w.rows
    room = torch.full((m, n + 2), 7.0, dtype=dtype, device="cuda")
    out = room[:, 1:n + 1]
    code = ops.lib("mx").fg_gemm_mxfp4_ext(x.data_ptr(), x.stride(0), w.data.data_ptr(), w.scales.data_ptr(), out.data_ptr(), int(dtype == torch.bfloat16),
                                           out.stride(0), 0, m, n, w.k, form, bn, splits, torch.cuda.current_stream().cuda_stream)
    assert code == 0 and (room[:, 0] == 7).all() and (room[:, n + 1:] == 7).all()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("form,bn,splits", [(1, 16, 1), (2, 16, 1), (2, 48, 3), (2, 112, 8), (2, 256, 1), (2, 256, 2), (3, 32, 1), (3, 96, 1), (3, 224, 1), (3, 256, 1)])
@pytest.mark.parametrize("m,n,k", [(1, 100, 32), (70, 129, 96), (40, 513, 1056), (300, 384, 2080), (777, 1000, 160)])
def test_every_kernel_at_every_width(form, bn, splits, m, n, k):
    x, (w, numbers) = _rows(m, k, m + n).cuda(), _matrix(n, k, n + k)
    want, slack = plain.product(x, numbers)
    plain.check(_named(x, w, form, bn, splits), want, slack)
    plain.check(_named(x, w, form, bn, splits, torch.bfloat16), want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("form,bn", [(2, 32), (3, 32), (3, 256)])
def test_many_tiles_a_processor(form, bn):
    """Every SM walks several tiles, of one stage of K and of many."""
    for m, n, k in ((1500, 1300, 32), (1500, 1300, 128), (900, 5000, 352), (2048, 4096, 1024)):
        x, (w, numbers) = _rows(m, k, m + n).cuda(), _matrix(n, k, n + k)
        want = (x.double() @ numbers.cuda().T).cpu()
        size = (x.double().abs() @ numbers.cuda().abs().T).cpu()
        plain.check(_named(x, w, form, bn), want, size * (2 * k / 16 + 32) * 2.0 ** -23)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 40001, 96), (8, 19999, 544), (3, 40000, 2048), (5, 4099, 14336), (2, 700, 40000), (20, 9001, 1056)])
def test_few_rows_over_many_units_and_long_rows(m, n, k):
    """Sizes for which the kernel for few rows takes units with fewer warps, and splits long rows over a cluster; the same call gives the same bits."""
    w, numbers = _matrix(n, k, 61)
    x = _rows(m, k, 62)
    odd = torch.zeros(m, k + 1, dtype=torch.bfloat16, device="cuda")                       # (rows that TMA cannot address, for more than eight)
    odd[:, :k] = x.cuda()
    want, slack = plain.product(x, numbers)
    for rows in (x.cuda(), odd[:, :k]):
        out = ops.gemm_mxfp4(rows, w, out_dtype=torch.float32)
        plain.check(out, want, slack)
        assert torch.equal(out, ops.gemm_mxfp4(rows, w, out_dtype=torch.float32))
        both = torch.full((m, n), 1.5, device="cuda")
        ops.gemm_mxfp4(rows, w, out=both, accumulate=True)
        assert torch.equal(both, out + 1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 16, 40, 130, 300])
def test_contraction_on_strided_rows(m):
    n, k = 333, 544
    wide = _rows(m, k + 24, 3).cuda()
    w, numbers = _matrix(n, k, 4)
    for at in (0, 8, 3):                                     # aligned, aligned further in, off the 16-byte grid
        x = wide[:, at:at + k]
        want, slack = plain.product(x, numbers)
        for dtype in (torch.bfloat16, torch.float32):
            room = torch.full((m + 2, n + 5), 7.0, dtype=dtype, device="cuda")
            ops.gemm_mxfp4(x, w, out=room[1:m + 1, 2:n + 2])
            plain.check(room[1:m + 1, 2:n + 2], want, slack)
            room[1:m + 1, 2:n + 2] = 7.0
            assert (room == 7.0).all()                       # nothing beside the output is touched
    odd = torch.zeros(m, k + 1, dtype=torch.bfloat16, device="cuda")
    odd[:, :k] = wide[:, :k]
    want, slack = plain.product(wide[:, :k], numbers)
    plain.check(ops.gemm_mxfp4(odd[:, :k], w), want, slack)
    same = wide[:1, :k].expand(m, k)                         # every row the same memory
    want, slack = plain.product(same, numbers)
    plain.check(ops.gemm_mxfp4(same, w), want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 12, 40, 200])
@pytest.mark.parametrize("low,high", [(0, 3), (0, 254), (128, 140), (190, 200)])
def test_contraction_over_exponents(m, low, high):
    """Exponents from the smallest to the largest; activations that keep every sum inside float32."""
    n, k = 140, 288
    data, e = plain.random_matrix(n, k, _gen(9), low, high)
    w, numbers = Mxfp4.from_exponents(data.cuda(), e.cuda()), plain.numbers(data, e)
    top = numbers.abs().max().item()
    x = (_rows(m, k, 10, loud=False).float() * min(1.0, 2.0 ** 100 / top)).bfloat16()
    if high == 254:                                          # codes of 2 and more under 2^127 are beyond bfloat16 and float32
        numbers = numbers.float().double()
        beyond = torch.isinf(numbers).any(1)
        got = ops.gemm_mxfp4(x.cuda(), w, out_dtype=torch.float32).cpu()
        assert not torch.isfinite(got[:, beyond]).any() or not beyond.any()
        keep = ~beyond
        want, slack = plain.product(x, numbers[keep])
        plain.check(got[:, keep], want, slack)
        return
    want, slack = plain.product(x, numbers)
    plain.check(ops.gemm_mxfp4(x.cuda(), w, out_dtype=torch.float32), want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 12, 40, 200])
def test_no_numbers_stay_in_their_row_and_column(m):
    n, k = 150, 160
    data, e = plain.random_matrix(n, k, _gen(11))
    e[7, 2] = 255
    w, numbers = Mxfp4.from_exponents(data.cuda(), e.cuda()), plain.numbers(data, e)
    x = _rows(m, k, 12)
    x[m // 2, 33] = float("nan")
    x[0, 5] = float("inf")
    got = ops.gemm_mxfp4(x.cuda(), w, out_dtype=torch.float32).cpu()
    want = x.double() @ numbers.T
    clean = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    ok = torch.isfinite(x.float()).all(1)
    assert ok.sum() == m - len({0, m // 2})
    cols = torch.arange(n) != 7
    assert clean[ok][:, cols].all()
    want, slack = plain.product(x[ok], numbers[cols])
    plain.check(got[ok][:, cols], want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 64, 32), (1, 2048, 2048), (7, 129, 96), (40, 300, 160), (128, 128, 128), (130, 257, 2080), (256, 512, 1024), (600, 200, 544)])
def test_contraction_of_two_quantised_operands(m, n, k):
    x = _rows(m, k, m + k)
    w, numbers = _matrix(n, k, n)
    q = ops.mxfp4_quantize(x.cuda())
    want, slack = plain.product(plain.rounded(x)[0], numbers)
    plain.check(ops.gemm_mxfp4_both(q, w), want, slack)
    got = ops.gemm_mxfp4_both(q, w, out_dtype=torch.float32)
    plain.check(got, want, slack)
    assert torch.equal(got, ops.gemm_mxfp4_both(q, w, out_dtype=torch.float32))
    res = torch.randn(m, n, generator=_gen(2)).cuda()
    room = torch.full((m, n + 3), 7.0, device="cuda")
    room[:, 1:n + 1] = res
    ops.gemm_mxfp4_both(q, w, out=room[:, 1:n + 1], accumulate=True)
    plain.check(room[:, 1:n + 1], want + res.double().cpu(), slack + 2.0 ** -24 * res.double().cpu().abs())
    assert (room[:, 0] == 7).all() and (room[:, n + 1:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 70, 352), (8, 64, 4096), (13, 128, 8192), (16, 40, 32768), (5, 33, 65536)])
def test_activations_of_any_range(m, n, k):
    """Few rows: numbers of one token that are many binades apart (the smallest beside the largest, where half precision cannot hold both),
    tokens of very different sizes, rows of zeros, K longer than what is staged at once."""
    g = _gen(m + k)
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-60, 30, (m, 1), generator=g).float())
    x[0] = 0
    x[1, ::7] = 0
    x[2, 5] = 2.0 ** 90                                      # under a weight of 0: nothing of it reaches the sums
    x[2, 40:] *= 2.0 ** -50
    x[m - 1] *= torch.exp2(torch.randint(-50, 10, (k,), generator=g).float())
    x = x.bfloat16()
    data, e = plain.random_matrix(n, k, g, 117, 123)
    data[:, 2] &= 15                                         # (number 5: the high half of byte 2)
    e[3], data[3] = 0, 0                                     # a row of zeros, as the quantiser makes it
    w, numbers = Mxfp4.from_exponents(data.cuda(), e.cuda()), plain.numbers(data, e)
    want, slack = plain.product(x, numbers)
    got = _named(x.cuda(), w, 1)
    plain.check(got, want, slack)
    assert (got[0] == 0).all() and (got[:, 3] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,bn,splits", [(1, 100, 32, 16, 1), (1, 128, 64, 16, 1), (5, 129, 128, 48, 1), (100, 130, 160, 112, 1), (128, 128, 256, 128, 1), (200, 500, 288, 208, 1),
                                             (256, 256, 512, 256, 1), (300, 384, 2080, 128, 1), (300, 384, 2080, 256, 1), (70, 300, 2048, 80, 3), (40, 100, 4096, 48, 8),
                                             (777, 1000, 1056, 256, 2), (2048, 4096, 1024, 256, 1), (1500, 5000, 96, 128, 1)])
def test_two_quantised_operands_at_every_width(m, n, k, bn, splits):
    w, numbers = _matrix(n, k, n)
    xm, xn = _matrix(m, k, m + 1, low=110, high=132)
    want = (xn.cuda() @ numbers.cuda().T).cpu()
    slack = (xn.cuda().abs() @ numbers.cuda().abs().T).cpu() * (2 * k / 16 + 32) * 2.0 ** -23
    out = torch.full((m, n + 2), 7.0, device="cuda")
    code = ops.lib("mx").fg_gemm_mxfp4_both_ext(xm.data.data_ptr(), xm.scales.data_ptr(), w.data.data_ptr(), w.scales.data_ptr(), out[:, 1:].data_ptr(), 0,
                                                n + 2, 0, m, n, k, bn, splits, torch.cuda.current_stream().cuda_stream)
    assert code == 0 and (out[:, 0] == 7).all() and (out[:, n + 1:] == 7).all()
    plain.check(out[:, 1:n + 1], want, slack)


def _runs(counts, before=0):
    return torch.tensor([before + sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("counts,n,k", [([1], 64, 32), ([0, 1, 0, 2], 65, 96), ([3, 0, 9, 1, 0, 17, 2, 0], 200, 160), ([130, 1, 0, 257, 64], 129, 512),
                                        ([0, 0, 0], 64, 64), ([1] * 40, 300, 2048), ([700, 0, 5], 384, 1056), ([0, 1, 2, 33, 0, 7, 1, 5], 260, 288),
                                        ([40, 0, 90, 3], 700, 160), ([0] * 1500 + [3, 1] + [0] * 10, 40, 64)])
def test_rows_grouped_by_expert(counts, n, k):
    P, X = sum(counts), len(counts)
    stack = [plain.random_matrix(n, k, _gen(100 + e)) for e in range(X)]
    w = Mxfp4.from_exponents(torch.stack([d for d, _ in stack]).cuda(), torch.stack([e for _, e in stack]).cuda())
    before, behind = 3, 6                                    # rows of no run in front and behind
    x = _rows(before + P + behind, k, 50)
    offsets = _runs(counts, before).cuda()
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((before + P + behind, n), 7.0, dtype=dtype, device="cuda")
        ops.gemm_mxfp4_grouped(x.cuda(), w, offsets, out=out)
        assert (out[:before] == 7).all() and (out[before + P:] == 7).all()
        at = before
        for c, (d, e) in zip(counts, stack):
            if c:
                want, slack = plain.product(x[at:at + c], plain.numbers(d, e))
                plain.check(out[at:at + c], want, slack)
            at += c
    again = torch.full_like(out, 7.0)
    ops.gemm_mxfp4_grouped(x.cuda(), w, offsets, out=again)
    assert torch.equal(out, again)
    odd = torch.zeros(x.shape[0], k + 1, dtype=torch.bfloat16, device="cuda")              # rows that TMA cannot address
    odd[:, :k] = x.cuda()
    other = torch.full_like(out, 7.0)
    ops.gemm_mxfp4_grouped(odd[:, :k], w, offsets, out=other)
    assert (other[:before] == 7).all() and (other[before + P:] == 7).all()
    at = before
    for c, (d, e) in zip(counts, stack):
        if c:
            want, slack = plain.product(x[at:at + c], plain.numbers(d, e))
            plain.check(other[at:at + c], want, slack)
        at += c
    if P:
        ops.gemm_mxfp4_grouped(x.cuda(), w, offsets, out=again, accumulate=True)
        assert torch.equal(again[before:before + P], 2 * out[before:before + P])


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [-4, 2, 4, 6], [0, 100, 200, 300], [7, 7, 7, 7], [9, 6, 3, 0]])
def test_offsets_that_name_no_rows_reach_none(offsets):
    """Offsets that fall, or leave the rows of x, are cut to them: nothing outside x and out is read or written."""
    n, k, M = 70, 64, 9
    stack = [plain.random_matrix(n, k, _gen(200 + e)) for e in range(3)]
    w = Mxfp4.from_exponents(torch.stack([d for d, _ in stack]).cuda(), torch.stack([e for _, e in stack]).cuda())
    x = _rows(M, k, 51)
    room = torch.full((M + 4, n), 7.0, device="cuda")
    ops.gemm_mxfp4_grouped(x.cuda(), w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out=room[2:M + 2])
    assert (room[:2] == 7).all() and (room[M + 2:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [9, 300, 1500])
def test_runs_that_overlap_many_times_reach_nothing_else(M):
    """Offsets that fall and rise again name every row by every other expert, far more tiles than rising offsets can: nothing outside out is written."""
    n, k, X = 70, 64, 64
    d, e = plain.random_matrix(n, k, _gen(210))
    w = Mxfp4.from_exponents(d.expand(X, *d.shape).cuda(), e.expand(X, *e.shape).cuda())
    x = _rows(M, k, 52)
    room = torch.full((M + 4, n), 7.0, device="cuda")
    offsets = torch.tensor([0, M] * (X // 2) + [0], dtype=torch.int32, device="cuda")
    ops.gemm_mxfp4_grouped(x.cuda(), w, offsets, out=room[2:M + 2])
    ops.raise_on_device_error("overlapping runs")
    assert (room[:2] == 7).all() and (room[M + 2:] == 7).all()
    want, slack = plain.product(x, plain.numbers(d, e))               # the matrices are alike: whoever wrote a row wrote this
    plain.check(room[2:M + 2], want, slack)


# ------------------------------------------------------------------------------ as a program uses them
@pytest.mark.gpu
def test_no_rows():
    w, _ = _matrix(65, 96, 1)
    x = torch.zeros(0, 96, dtype=torch.bfloat16, device="cuda")
    assert ops.gemm_mxfp4(x, w).shape == (0, 65)
    assert ops.gemm_mxfp4_both(ops.mxfp4_quantize(x), w).shape == (0, 65)
    stack = Mxfp4(w.data[None], w.scales[None])
    assert ops.gemm_mxfp4_grouped(x, stack, torch.zeros(2, dtype=torch.int32, device="cuda")).shape == (0, 65)


def _block(x, table, up, down, experts, offsets, tokens):
    """A piece of a decoder: lookup, a feed-forward with 4-bit weights into the residual stream, experts, and a product of two quantised operands."""
    stream = ops.mxfp4_rows(table, tokens, scale=2.0)
    h = ops.gemm_mxfp4(x, up)
    ops.gemm_mxfp4(h, down, out=stream, accumulate=True)
    xs = stream.bfloat16()
    ops.gemm_mxfp4_grouped(xs, experts, offsets, out=stream, accumulate=True)
    logits = ops.gemm_mxfp4_both(ops.mxfp4_quantize(stream), table, out_dtype=torch.float32)
    return stream, logits


def _block_inputs(m, seed):
    E, F, V = 160, 352, 300
    table, t64 = _matrix(V, E, seed, low=118, high=121)
    up, u64 = _matrix(F, E, seed + 1, low=118, high=121)
    down, d64 = _matrix(E, F, seed + 2, low=118, high=121)
    ex = [plain.random_matrix(E, E, _gen(seed + 3 + e), 118, 121) for e in range(3)]
    experts = Mxfp4.from_exponents(torch.stack([d for d, _ in ex]).cuda(), torch.stack([e for _, e in ex]).cuda())
    cut = [0, m // 3, m // 3, m]
    tokens = torch.randint(0, V, (m,), generator=_gen(seed), dtype=torch.int32)
    x = _rows(m, E, seed + 9, loud=False)
    return (x, tokens, (t64, u64, d64, [plain.numbers(d, e) for d, e in ex], cut)), (
        x.cuda(), table, up, down, experts, torch.tensor(cut, dtype=torch.int32, device="cuda"), tokens.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 24, 150])
def test_a_run_of_them(m):
    (x, tokens, (t64, u64, d64, ex, cut)), args = _block_inputs(m, 60)
    stream, logits = _block(*args)
    want, slack = plain.product(x, u64)
    plain.check(ops.gemm_mxfp4(args[0], args[2]), want, slack)
    h = ops.gemm_mxfp4(args[0], args[2]).double().cpu()
    s, s_slack = plain.product(h, d64)
    s = s + 2 * t64[tokens.long()]
    mid = (2 * t64[tokens.long()]).float().cuda()
    ops.gemm_mxfp4(ops.gemm_mxfp4(args[0], args[2]), args[3], out=mid, accumulate=True)
    plain.check(mid, s, s_slack)
    xs = mid.bfloat16()
    for e in range(3):
        a, b = cut[e], cut[e + 1]
        if b > a:
            want, slack = plain.product(xs[a:b].cpu(), ex[e])
            plain.check(stream[a:b], want + mid[a:b].double().cpu(), slack)
    q, _ = plain.rounded(stream)
    want, slack = plain.product(q, t64)
    plain.check(logits, want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 24, 150])
def test_on_another_stream_and_recorded(m):
    _, args = _block_inputs(m, 70)
    want = _block(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs recorded side by side, replayed in turn on changed inputs
    other = _block_inputs(m, 90)[1]
    graphs, outs = [], []
    for a in (args, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_block(*a))
        graphs.append(graph)
    expected_other = _block(*other)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want)) and all(torch.equal(a, b) for a, b in zip(outs[1], expected_other))
    args[0].copy_(other[0])
    expected = _block(*args)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], expected))


@pytest.mark.gpu
def test_two_calls_at_once():
    """The same operator on two streams at a time: nothing is shared between calls."""
    sets = [_block_inputs(m, 110 + m)[1] for m in (40, 200)]
    want = [_block(*a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for s, a in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(_block(*a))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, want[i % 2]))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 2048, 2048), (12, 28672, 4096), (40, 2048, 4096), (200, 8192, 2048)])
def test_beside_a_stream_that_keeps_memory_busy(m, n, k):
    """Every form starts and ends many times while another stream quantises and reads large matrices: the same bits as alone."""
    w, _ = _matrix(n, k, 71)
    stack = Mxfp4(w.data.view(4, n // 4, k // 2), w.scales.view(4, n // 512, -1, 32, 4, 4))
    x, other = _rows(m, k, 72).cuda(), torch.randn(8192, 4096, device="cuda")
    q, offsets = ops.mxfp4_quantize(x), torch.tensor([0, m // 3, m // 3, m, m], dtype=torch.int32, device="cuda")
    calls = [lambda: ops.gemm_mxfp4(x, w), lambda: ops.gemm_mxfp4_both(q, w), lambda: ops.gemm_mxfp4_grouped(x, stack, offsets)]
    calls += [lambda f=f, b=b, z=z: _named(x, w, f, b, z) for f, b, z in [(2, 16, 1), (2, 48, 2), (2, 256, 1), (3, 32, 1), (3, 256, 1)] if z == 1 or n <= 2048]
    alone = [c().clone() for c in calls]
    beside, mine = torch.cuda.Stream(), torch.cuda.Stream()
    beside.wait_stream(torch.cuda.current_stream())
    mine.wait_stream(torch.cuda.current_stream())
    for _ in range(15):
        with torch.cuda.stream(beside):
            for _ in range(4):
                ops.mxfp4_rows(ops.mxfp4_quantize(other))
        with torch.cuda.stream(mine):
            for c, want in zip(calls, alone):
                assert torch.equal(c(), want)
    torch.cuda.synchronize()
    ops.raise_on_device_error("beside another stream")


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["tiles", "tiles split", "pairs", "both"])
def test_a_wait_that_runs_out_ends_the_kernel_and_the_next_is_correct(which):
    """The first copy of tokens is left out and waits are shortened to about a millisecond: the kernel gives up, raises its error flag, frees its tensor
    memory and returns."""
    import time
    from ctypes import c_int, c_longlong
    m, n, k = 100, 300, 2048
    bn = 96 if which == "pairs" else 112
    w, numbers = _matrix(n, k, 8)
    x = _rows(m, k, 9)
    q, xd = ops.mxfp4_quantize(x.cuda()), x.cuda()

    def call():
        if which == "both":
            return ops.gemm_mxfp4_both(q, w, out_dtype=torch.float32)
        return _named(xd, w, 3 if which == "pairs" else 2, bn, 4 if which == "tiles split" else 1).clone()

    error, hook = ops.lib("mx").fg_gemm_mxfp4_error, ops.lib("mx").fg_gemm_mxfp4_test_hook
    hook.argtypes, hook.restype = [c_longlong, c_int], c_int
    want, slack = plain.product(plain.rounded(x)[0] if which == "both" else x, numbers)
    before = call()
    plain.check(before, want, slack)
    assert error() == 0
    try:
        assert hook(2_000_000, 1) == 0
        t0 = time.time()
        if which == "both":
            call()
        else:
            out = torch.empty(m, n, device="cuda")
            ops.lib("mx").fg_gemm_mxfp4_ext(xd.data_ptr(), k, w.data.data_ptr(), w.scales.data_ptr(), out.data_ptr(), 0, n, 0, m, n, k, 3 if which == "pairs" else 2,
                                            bn, 4 if which == "tiles split" else 1, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert time.time() - t0 < 2.0
        with pytest.raises(KernelError, match="wait ran out"):
            ops.raise_on_device_error("test")
    finally:
        assert hook(0, 0) == 0
    assert error() == 0
    assert torch.equal(call(), before) and error() == 0
