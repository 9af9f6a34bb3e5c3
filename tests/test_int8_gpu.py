"""Rows as 8-bit integers and their grouped products, against their definitions in 64 bits.

quantize_rows is defined exactly: 127 x / max|x| to the nearest integer, ties to even, and the fp32 quotient max|x| / 127.  In 64 bits the quotient of
a 32-bit number times 127 by another is exact where it is a tie, and otherwise further from one than its rounding, so that
integers and scales are equal.

swiglu_quantize's silu(gate) * up is computed in fp32: the exponential is off by two units in the last place, the sum, the quotient and the
product by one each at most, together below 2^-21 of the value.  So scales are off by that and a rounding, below 2^-20, and a value
that 127 / max takes to at most 127 moves by less than 127 * 2^-19 = 2^-12 steps: integers are within a half and 2^-12 of what they round.

gmm_int8's sums are exact; they are rounded to fp32, multiplied twice and rounded to the type: off by 3 * 2^-24 and half a step of the
type (bf16 2^-8, fp16 2^-11 of the value; below fp16's normal range half of 2^-24)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ROUNDING = {torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25)}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from grouped_gemm import ops as _ops
    return _ops


def _announce(*what):
    print("[case]", *what, flush=True)


def _quantized(x):
    """By the definition, of finite rows."""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    q = torch.round(127.0 * x / torch.where(most > 0, most, torch.ones_like(most)))
    return q.to(torch.int8), (most / 127.0).float().squeeze(-1)


def _check_rows(ops, x, what, row_index=None):
    """x: on the CPU."""
    got = ops.quantize_rows(x.cuda(), None if row_index is None else row_index.cuda())
    rows = x if row_index is None else x[row_index.long()]
    values, scales = _quantized(rows)
    assert got.values.dtype == torch.int8 and got.scales.dtype == torch.float32
    assert got.values.shape == rows.shape and got.scales.shape == rows.shape[:-1], what
    assert torch.equal(got.scales.cpu(), scales), what
    assert torch.equal(got.values.cpu(), values), (what, int((got.values.cpu() != values).sum()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (5, 63), (130, 65), (9, 512), (7, 513), (6, 1024), (5, 1025), (3, 2047), (66, 2048),
                                       (3, 2049), (70, 4096), (2, 4099), (3, 8192), (2, 8193), (2, 16384), (2, 16391), (1, 70001)])
def test_rows_are_the_nearest_integers(ops, dtype, rows, cols):
    _announce("rows", dtype, rows, cols)
    g = torch.Generator().manual_seed(rows * 100003 + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
    _check_rows(ops, x.to(dtype), (dtype, rows, cols))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_even_integer(ops, dtype):
    _announce("ties", dtype)
    halves = torch.arange(-126.5, 127.0, 0.5)
    rows = torch.stack([torch.cat([halves, torch.tensor([127.0])]) * scale for scale in (1.0, 2.0, 2.0 ** -9, 8.0)])
    rows = torch.cat([rows, rows.flip(1)])
    assert torch.equal(rows.to(dtype).float(), rows) or dtype == torch.bfloat16
    _check_rows(ops, rows.to(dtype), ("ties", dtype))
    # ... and next to them
    if dtype == torch.float32:
        near = torch.cat([torch.nextafter(rows, torch.tensor(INF)), torch.nextafter(rows, torch.tensor(-INF))])
        near[:, 0] = 127.0 * 8
        _check_rows(ops, near, "next to ties")
        most = torch.tensor([[3.7], [1.1], [97.3], [5e-3]])   # ties that no float is: the two floats around each
        t = (halves * most / 127.0).float()
        near = torch.cat([t, torch.nextafter(t, torch.tensor(INF)), torch.nextafter(t, torch.tensor(-INF)), most], 1)
        _check_rows(ops, near, "around ties")
    # small integers and few bits: many quotients are ties
    g = torch.Generator().manual_seed(1)
    few = torch.randint(-254, 255, (200, 300), generator=g).float()
    few[:, 0] = 254.0
    _check_rows(ops, few.to(dtype), ("few bits", dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_any_size(ops, dtype):
    _announce("sizes", dtype)
    g = torch.Generator().manual_seed(2)
    info = torch.finfo(dtype)
    x = torch.randn(8, 600, generator=g).clamp(-3, 3)
    x = x / x.abs().amax(1, keepdim=True)
    factors = torch.tensor([info.max, info.tiny, info.tiny * 2 ** -4, info.tiny * info.eps * 3, info.tiny * info.eps, 1e-20, 1.0, 0.0], dtype=torch.float64)
    _check_rows(ops, (x.double() * factors.unsqueeze(1)).to(dtype), ("sizes", dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [5, 700, 5000])
def test_rows_with_infinities_and_nan(ops, dtype, cols):
    _announce("odd values", dtype, cols)
    x = torch.randn(6, cols)
    x[1, 3], x[1, 1] = INF, -INF
    x[2, 2] = NAN
    x[3, 0], x[3, 4] = NAN, INF
    x[4, cols - 1] = -NAN
    got = ops.quantize_rows(x.to(dtype).cuda())
    q, s = got.values.cpu(), got.scales.cpu()
    want, scales = _quantized(x[[0, 5]].to(dtype))
    assert torch.equal(q[[0, 5]], want) and torch.equal(s[[0, 5]], scales)
    assert s[1] == INF and all(math.isnan(s[i]) for i in (2, 3, 4))
    infinite = torch.zeros(cols, dtype=torch.int8)
    infinite[3], infinite[1] = 127, -127
    assert torch.equal(q[1], infinite)
    # products of such rows are not finite, of the others not touched
    b = ops.quantize_rows(torch.randn(1, 16, cols, device="cuda"))
    out = ops.gmm_int8(got.values, got.scales, b.values, b.scales, torch.tensor([6])).cpu()
    assert torch.isfinite(out[[0, 5]]).all() and not torch.isfinite(out[1:5]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [33, 1000, 4096])
def test_rows_through_an_index(ops, dtype, cols):
    _announce("index", dtype, cols)
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(50, cols, generator=g).to(dtype)
    _check_rows(ops, x, "index", torch.randint(50, (173,), generator=g, dtype=torch.int32))
    _check_rows(ops, x, "all the same", torch.full((20,), 7, dtype=torch.int32))
    _check_rows(ops, x, "no rows", torch.empty(0, dtype=torch.int32))
    # numbers that name no row: zeros
    index = torch.tensor([3, -1, 50, 2 ** 31 - 1, -2 ** 31, 49], dtype=torch.int32)
    got = ops.quantize_rows(x.cuda(), index.cuda())
    want, scales = _quantized(x[[3, 49]])
    assert torch.equal(got.values[[0, 5]].cpu(), want) and torch.equal(got.scales[[0, 5]].cpu(), scales)
    assert not got.values[1:5].any() and not got.scales[1:5].any()
    none = ops.quantize_rows(x[:0].cuda(), index.cuda())
    assert none.values.shape == (6, cols) and not none.values.any() and not none.scales.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_weights_and_of_views(ops, dtype):
    _announce("views", dtype)
    g = torch.Generator().manual_seed(3)
    _check_rows(ops, torch.randn(3, 20, 77, generator=g).to(dtype), "three dimensions")
    _check_rows(ops, torch.randn(77, generator=g).to(dtype), "one dimension")
    _check_rows(ops, torch.randn(0, 77, generator=g).to(dtype), "no rows")
    wide = torch.randn(40, 900, generator=g).to(dtype)
    for first, last in ((0, 500), (1, 900), (3, 40), (8, 136)):
        got = ops.quantize_rows(wide.cuda()[:, first:last])
        want, scales = _quantized(wide[:, first:last])
        assert torch.equal(got.values.cpu(), want) and torch.equal(got.scales.cpu(), scales), (first, last)
        got = ops.quantize_rows(wide.cuda()[::3, first:last], torch.tensor([2, 0], dtype=torch.int32, device="cuda"))
        assert torch.equal(got.values.cpu(), want[[6, 0]]), (first, last)


def _check_swiglu(ops, gate_up, what):
    """Of finite results; gate_up on the CPU."""
    got = ops.swiglu_quantize(gate_up.cuda())
    gate, up = gate_up.double().chunk(2, -1)
    h = gate / (1.0 + torch.exp(-gate)) * up
    most = h.abs().amax(-1)
    scales = got.scales.double().cpu()
    assert ((scales - most / 127.0).abs() <= 2.0 ** -20 * most / 127.0 + 2.0 ** -149).all(), what
    off = (got.values.double().cpu() * scales.unsqueeze(-1) - h).abs()
    assert (off <= (0.5 + 2.0 ** -12) * (most / 127.0).unsqueeze(-1) + 2.0 ** -142).all(), what
    assert got.values.shape == h.shape and got.scales.shape == h.shape[:-1]
    largest = torch.where(most > 2.0 ** -120, got.values.abs().amax(-1).cpu().double(), torch.full_like(most, 127.0))
    assert (largest == 127).all(), what


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ffn", [(1, 1), (3, 9), (1, 1408), (5, 511), (4, 2047), (3, 2048), (2, 14336), (2, 20001), (300, 96)])
def test_gated_rows(ops, dtype, rows, ffn):
    _announce("gated", dtype, rows, ffn)
    g = torch.Generator().manual_seed(ffn)
    _check_swiglu(ops, (2 * torch.randn(rows, 2 * ffn, generator=g)).to(dtype), (dtype, rows, ffn))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(2048, 515), (2049, 515), (2049, 1030), (2048, 2040), (2051, 2040), (1024, 2056), (1025, 2056), (1025, 4095), (700, 5000), (300, 9001)])
def test_many_rows(ops, dtype, rows, cols):
    """Either side of the numbers of rows at which other kernels take them, of rows and of rows that an index names or not."""
    _announce("many rows", dtype, rows, cols)
    g = torch.Generator().manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)
    _check_rows(ops, x, (dtype, rows, cols))
    index = torch.randint(-20, rows + 20, (rows,), generator=g).to(torch.int32)
    got = ops.quantize_rows(x.cuda(), index.cuda())
    named = (index >= 0) & (index < rows)
    values, scales = _quantized(x[index.clamp(0, rows - 1).long()])
    assert torch.equal(got.values.cpu(), torch.where(named.unsqueeze(1), values, 0)) and torch.equal(got.scales.cpu(), torch.where(named, scales, 0.0))
    half = cols // 2
    _check_swiglu(ops, (1.5 * torch.randn(rows, 2 * half, generator=g)).to(dtype), (dtype, rows, half))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_rows_of_any_size(ops, dtype):
    _announce("gated sizes", dtype)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 400, generator=g)
    x[0] *= 60      # (exponentials past a float's range)
    x[1] *= 1e-4
    x[2, 200:] = 0.0
    x[3, :200] = -80.0
    x[4, :200] = -30.0
    _check_swiglu(ops, x.to(dtype)[[0, 1, 4, 5]], "sizes")
    got = ops.swiglu_quantize(x.to(dtype).cuda())
    assert not got.values[2].any() and got.scales[2] == 0
    view = torch.randn(7, 700, generator=g).to(dtype)
    got = ops.swiglu_quantize(view.cuda()[:, 5:305])
    whole = ops.swiglu_quantize(view[:, 5:305].contiguous().cuda())
    assert torch.equal(got.values, whole.values) and torch.equal(got.scales, whole.scales)
    x[1, 7] = NAN
    got = ops.swiglu_quantize(x.to(dtype).cuda())
    assert math.isnan(got.scales[1]) and torch.isfinite(got.scales[[0, 3, 4, 5]]).all()


# ------------------------------------------------------------------ grouped products

def _operands(rows, experts, hidden_in, hidden_out, seed):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-128, 128, (rows, hidden_in), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (experts, hidden_out, hidden_in), generator=g, dtype=torch.int8)
    return a, torch.rand(rows, generator=g) / 64 + 1e-3, b, torch.rand(experts, hidden_out, generator=g) / 64 + 1e-3


def _product(a, a_scales, b, b_scales, sizes):
    """In 64 bits; rows behind the last expert's are NaN."""
    out = torch.full((a.shape[0], b.shape[1]), NAN, dtype=torch.float64)
    start = 0
    for e, n in enumerate(sizes):
        if n > 0:
            out[start:start + n] = (a[start:start + n].double() @ b[e].double().t()) * a_scales[start:start + n].double().unsqueeze(1) * b_scales[e].double()
        start += n
    return out


def _check_close(got, want, dtype, what):
    half, least = ROUNDING[dtype]
    got = got.double().cpu()
    beyond = want.abs() > (1 + half) * torch.finfo(dtype).max   # (more than the type holds: an infinity of its sign)
    assert torch.equal(got[beyond], torch.sign(want[beyond]) * INF), what
    held = ~torch.isnan(want) & ~beyond
    off = (got - want).abs()[held] - ((half + 3 * 2.0 ** -24) * want.abs()[held] + least)
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))


def _run(ops, a, a_scales, b, b_scales, sizes, dtype, on_device, c=None):
    batch_sizes = torch.tensor(sizes, dtype=torch.int64)
    return ops.gmm_int8(a.cuda(), a_scales.cuda(), b.cuda(), b_scales.cuda(), batch_sizes.cuda() if on_device else batch_sizes, dtype=dtype, c=c)


SIZES = [
    # few rows to a group, one to four windows of each kind; every alignment of the depth
    ([1], 64, 64), ([1], 1, 1), ([2, 0, 1], 15, 3), ([5], 16, 65), ([3, 1], 17, 64), ([16], 127, 63), ([17, 16, 0, 1], 128, 129), ([33], 130, 31),
    ([8, 9, 7], 1021, 100), ([20, 30, 10], 514, 70), ([64, 65, 63], 259, 130), ([200, 1], 1023, 17), ([0, 0, 3, 0], 640, 64), ([4], 4096, 512),
    ([1, 1], 8192, 256), ([2], 14336, 128), ([40, 3], 6000, 64),
    # tiles: short, small and full ones, ragged rows
    ([100, 60, 0, 130], 256, 264), ([300, 700, 5], 512, 1024), ([129, 40, 257], 1040, 520), ([2000, 48, 1000], 2048, 2048), ([513], 4096, 8),
    ([40] * 24, 112, 136), ([1500, 1700], 16, 256), ([700], 16384, 128), ([1024, 1024, 1024, 1024], 1408, 2816),
    # ... that the streaming kernel does not take
    ([300, 150], 250, 130), ([500], 513, 1001), ([333, 0, 400], 2047, 263),
    # ... and of any width, whole tiles and pieces of the depth
    ([300, 700, 5], 512, 1021), ([100, 60, 0, 130], 256, 263), ([700], 16384, 121), ([513], 4096, 9), ([2000, 48, 1000], 2048, 2047), ([40] * 24, 112, 129),
    ([257, 300], 4112, 1), ([600], 8192, 514),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,hidden_in,hidden_out", SIZES, ids=lambda v: str(v)[:24])
def test_products_are_exact_sums_rounded_once(ops, dtype, sizes, hidden_in, hidden_out):
    _announce("product", dtype, sizes, hidden_in, hidden_out)
    rows = sum(sizes)
    a, sa, b, sb = _operands(rows, len(sizes), hidden_in, hidden_out, hidden_in + rows)
    want = _product(a, sa, b, sb, sizes)
    got = [_run(ops, a, sa, b, sb, sizes, dtype, on_device) for on_device in (True, False)]
    assert got[0].dtype == dtype and got[0].shape == (rows, hidden_out)
    _check_close(got[0], want, dtype, (sizes, hidden_in, hidden_out))
    assert torch.equal(got[0], got[1])


def _misaligned(t, elements):
    """A contiguous copy that begins `elements` behind a boundary."""
    buffer = torch.empty(t.numel() + 64, dtype=t.dtype, device="cuda")
    view = buffer[elements:elements + t.numel()].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.parametrize("sizes,hidden_in,hidden_out", [([5, 1], 256, 70), ([3, 20], 1024, 64), ([300, 200], 512, 264), ([700], 1040, 128), ([90, 40], 30, 33)])
def test_operands_on_any_boundary(ops, sizes, hidden_in, hidden_out):
    _announce("boundaries", sizes, hidden_in, hidden_out)
    rows = sum(sizes)
    a, sa, b, sb = _operands(rows, len(sizes), hidden_in, hidden_out, 7)
    want = _product(a, sa, b, sb, sizes)
    batch_sizes = torch.tensor(sizes).cuda()
    for off_a, off_b, off_c in ((1, 0, 0), (0, 3, 1), (2, 2, 2), (5, 15, 3), (8, 4, 4), (0, 0, 1)):
        buffer = torch.full((rows * hidden_out + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
        c = buffer[off_c:off_c + rows * hidden_out].view(rows, hidden_out)
        out = ops.gmm_int8(_misaligned(a, off_a), _misaligned(sa, 1), _misaligned(b, off_b), _misaligned(sb, 3), batch_sizes, c=c)
        assert out.data_ptr() == c.data_ptr()
        _check_close(out, want, torch.bfloat16, (off_a, off_b, off_c))
        assert (buffer[:off_c] == 7).all() and (buffer[off_c + rows * hidden_out:] == 7).all()


@pytest.mark.parametrize("sizes,hidden_in,hidden_out", [([1, 2], 4095, 130), ([16], 4097, 65), ([17, 9, 20], 4098, 600), ([40, 33], 2047, 1023), ([64, 50], 6001, 200), ([3] * 9, 2303, 64),
                                                        ([1], 14335, 63)] + [([n], 2049, 700) for n in (24, 25, 32, 33, 64, 65)] + [([n], 1040, 700) for n in (24, 25, 32, 33, 64, 65)])
def test_deep_products_of_few_rows_on_any_boundary(ops, sizes, hidden_in, hidden_out):
    """Steps of the depth in the kernel's loop, of windows of 16, 32 and 64 rows; one group either side of the rows at which tiles take it."""
    _announce("deep", sizes, hidden_in, hidden_out)
    rows = sum(sizes)
    a, sa, b, sb = _operands(rows, len(sizes), hidden_in, hidden_out, rows + hidden_in)
    want = _product(a, sa, b, sb, sizes)
    batch_sizes = torch.tensor(sizes).cuda()
    for off_a, off_b in ((0, 0), (1, 2), (3, 0), (4, 8)):
        out = ops.gmm_int8(_misaligned(a, off_a), sa.cuda(), _misaligned(b, off_b), sb.cuda(), batch_sizes, dtype=torch.float16)
        _check_close(out, want, torch.float16, (off_a, off_b))


@pytest.mark.parametrize("hidden_in,hidden_out", [(64, 64), (256, 1024), (63, 65), (4096, 128)])
@pytest.mark.parametrize("sizes", [[3, 0, 2], [40, 30, 0, 7], [300, 200, 100], [2000]])
def test_rows_behind_the_last_group_keep_what_they_hold(ops, sizes, hidden_in, hidden_out):
    _announce("behind", sizes, hidden_in, hidden_out)
    rows = sum(sizes) + 37
    a, sa, b, sb = _operands(rows, len(sizes), hidden_in, hidden_out, 9)
    want = _product(a, sa, b, sb, sizes)
    for on_device in (True, False):
        c = torch.full((rows, hidden_out), 3.0, dtype=torch.float16, device="cuda")
        out = _run(ops, a, sa, b, sb, sizes, torch.float16, on_device, c=c)
        _check_close(out, want, torch.float16, sizes)
        assert (c[sum(sizes):] == 3).all()


def test_largest_sums(ops):
    """-128 * -128 over the largest depth, and just below zero; and the scales' own range."""
    depth = 131071
    a = torch.full((3, depth), -128, dtype=torch.int8)
    a[1] = 127
    b = torch.full((2, 9, depth), -128, dtype=torch.int8)
    sa, sb = torch.tensor([1.0, 2.0 ** -100, 2.0 ** 100]), torch.full((2, 9), 1.0)
    sb[1] = 2.0 ** -30
    for sizes in ([2, 1], [0, 3], [3, 0]):
        _check_close(_run(ops, a, sa, b, sb, sizes, torch.bfloat16, True), _product(a, sa, b, sb, sizes), torch.bfloat16, sizes)
    a, b = a[:, :131056].repeat(30, 1).contiguous(), b[:, :, :131056].contiguous()   # (the streaming kernel)
    sa = torch.ones(90)
    _check_close(_run(ops, a, sa, b, sb, [50, 40], torch.bfloat16, True), _product(a, sa, b, sb, [50, 40]), torch.bfloat16, "stream")


def test_no_depth_no_rows_no_columns(ops):
    sizes = torch.tensor([2, 0, 1])
    out = ops.gmm_int8(torch.empty(3, 0, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"), torch.empty(3, 5, 0, dtype=torch.int8, device="cuda"),
                       torch.ones(3, 5, device="cuda"), sizes)
    assert out.shape == (3, 5) and not out.any()
    for on_device in (True, False):
        a, sa, b, sb = _operands(0, 3, 64, 40, 1)
        assert _run(ops, a, sa, b, sb, [0, 0, 0], torch.bfloat16, on_device).shape == (0, 40)
        a, sa, b, sb = _operands(4, 3, 64, 0, 1)
        assert _run(ops, a, sa, b, sb, [1, 2, 1], torch.bfloat16, on_device).shape == (4, 0)
        a, sa, b, sb = _operands(4, 0, 64, 8, 1)
        c = torch.full((4, 8), 2.0, dtype=torch.bfloat16, device="cuda")
        assert (_run(ops, a, sa, b, sb, [], torch.bfloat16, on_device, c=c) == 2).all()
        a, sa, b, sb = _operands(5, 2, 64, 8, 1)   # (sizes of zero, rows behind)
        c = torch.full((5, 8), 2.0, dtype=torch.bfloat16, device="cuda")
        assert (_run(ops, a, sa, b, sb, [0, 0], torch.bfloat16, on_device, c=c) == 2).all()


@pytest.mark.parametrize("on_device", [True, False])
@pytest.mark.parametrize("rows", [0, 5, 700])
def test_no_experts_on_any_boundary(ops, rows, on_device):
    """Nothing is named, nothing is read: rows of c stay, whatever the depth."""
    for hidden_in, hidden_out in ((63, 8), (64, 8), (15, 9)):
        a, sa, b, sb = _operands(rows, 0, hidden_in, hidden_out, 1)
        c = torch.full((rows, hidden_out), 2.0, dtype=torch.bfloat16, device="cuda")
        assert (_run(ops, a, sa, b, sb, [], torch.bfloat16, on_device, c=c) == 2).all()
        assert _run(ops, a, sa, b, sb, [], torch.float16, on_device).shape == (rows, hidden_out)


@pytest.mark.parametrize("experts,rows", [(513, 700), (700, 40000), (1500, 1500), (600, 20)])
def test_more_groups_than_a_launch_takes(ops, experts, rows):
    _announce("groups", experts, rows)
    g = torch.Generator().manual_seed(experts)
    sizes = torch.bincount(torch.randint(experts, (rows,), generator=g), minlength=experts)
    a, sa, b, sb = _operands(rows, experts, 48, 24, 4)
    want = torch.empty(rows, 24, dtype=torch.float64)
    of_row = torch.repeat_interleave(torch.arange(experts), sizes)
    want = torch.matmul(b[of_row].double(), a.double().unsqueeze(2)).squeeze(2) * sa.double().unsqueeze(1) * sb[of_row].double()
    for on_device in (True, False):
        _check_close(_run(ops, a, sa, b, sb, sizes.tolist(), torch.bfloat16, on_device), want, torch.bfloat16, (experts, rows))


@pytest.mark.parametrize("hidden_in,hidden_out,rows", [(64, 40, 30), (256, 512, 900), (63, 40, 300)])
def test_wild_device_sizes_are_clamped_and_reported(ops, hidden_in, hidden_out, rows):
    from grouped_gemm_amd import backend
    _announce("wild sizes", hidden_in, hidden_out, rows)
    a, sa, b, sb = _operands(rows, 4, hidden_in, hidden_out, 3)
    backend.backend.size_status(torch.device("cuda", 0))
    for sizes, taken, status in (([5, 2, rows, 9], [5, 2, rows - 7, 0], True), ([-3, 4, 2, 0], [0, 4, 2, 0], True), ([2 ** 62, 2 ** 62, 1, 1], [rows, 0, 0, 0], True),
                                 ([1, 2, 3, 4], [1, 2, 3, 4], False), ([-2 ** 63, 1, 2 ** 63 - 1, -1], [0, 1, rows - 1, 0], True)):
        c = torch.full((rows, hidden_out), 9.0, dtype=torch.bfloat16, device="cuda")
        out = _run(ops, a, sa, b, sb, sizes, torch.bfloat16, True, c=c)
        _check_close(out, _product(a, sa, b, sb, taken), torch.bfloat16, sizes)
        assert (out[sum(taken):] == 9).all()
        assert bool(backend.backend.size_status(torch.device("cuda", 0))) == status, sizes
        if status:
            with pytest.raises(RuntimeError):
                _run(ops, a, sa, b, sb, sizes, torch.bfloat16, False)


@pytest.mark.parametrize("sizes,hidden_in,hidden_out", [([2, 1], 14336, 128), ([40, 9, 30], 2048, 192), ([700], 8192, 128), ([600, 300], 513, 64)])
def test_the_same_bits_on_every_call_and_stream(ops, sizes, hidden_in, hidden_out):
    _announce("repeats", sizes, hidden_in, hidden_out)
    a, sa, b, sb = (v.cuda() for v in _operands(sum(sizes), len(sizes), hidden_in, hidden_out, 11))
    batch_sizes = torch.tensor(sizes).cuda()
    first = ops.gmm_int8(a, sa, b, sb, batch_sizes)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.gmm_int8(a, sa, b, sb, batch_sizes))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("sizes,hidden_in,hidden_out", [([2, 1, 0], 4096, 128), ([30, 9, 1], 1024, 64), ([300, 700, 200], 512, 256), ([300, 0, 233], 511, 63)])
def test_captured_and_replayed(ops, sizes, hidden_in, hidden_out):
    """A chain from rows to rows, replayed with other rows and other sizes, with eager work between."""
    _announce("graph", sizes, hidden_in, hidden_out)
    rows, experts = sum(sizes), len(sizes)
    x = torch.randn(rows, hidden_in, device="cuda", dtype=torch.bfloat16)
    b = ops.quantize_rows(torch.randn(experts, 2 * hidden_out, hidden_in, device="cuda"))
    batch_sizes = torch.tensor(sizes).cuda()

    def chain():
        q = ops.quantize_rows(x)
        return ops.swiglu_quantize(ops.gmm_int8(q.values, q.scales, b.values, b.scales, batch_sizes, dtype=torch.float16))

    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    for n in range(4):
        x.copy_(torch.randn_like(x) * (n + 1))
        batch_sizes.copy_(torch.tensor(sizes[n % experts:] + sizes[:n % experts]))
        graph.replay()
        torch.cuda.synchronize()
        got = out.values.clone(), out.scales.clone()
        eager = chain()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager.values) and torch.equal(got[1], eager.scales), n


def test_more_columns_than_a_launch_for_few_rows_takes(ops):
    """Windows of rows times strips of columns past 2^24, a limit of the kernel for few rows, on the streaming one."""
    _announce("wide")
    experts, hidden_in, hidden_out = 512, 16, 1_725_440
    sizes = torch.full((experts,), 8)
    sizes[::100] += 1
    rows = int(sizes.sum())   # (8 to an expert and a few more)
    b = torch.empty(experts, hidden_out, hidden_in, dtype=torch.int8, device="cuda").random_(-128, 128)   # 14 GB, and as much of results
    sb = torch.rand(experts, hidden_out, device="cuda") / 64 + 1e-3
    a = torch.empty(rows, hidden_in, dtype=torch.int8, device="cuda").random_(-128, 128)
    sa = torch.rand(rows, device="cuda") / 64 + 1e-3
    got = ops.gmm_int8(a, sa, b, sb, sizes.cuda())
    ends = sizes.cumsum(0)
    for e in (0, 1, 255, 300, 511):
        for r in (int(ends[e] - sizes[e]), int(ends[e]) - 1):
            for at in (slice(0, 300), slice(hidden_out // 2, hidden_out // 2 + 300), slice(hidden_out - 300, hidden_out)):
                want = ((b[e, at].double() * a[r].double()).sum(1) * sa[r].double() * sb[e, at].double()).cpu()
                _check_close(got[r, at], want, torch.bfloat16, (e, r))


def test_offsets_past_32_bits(ops):
    """More than 4 GiB of weights, and more than 4 GiB of rows."""
    _announce("large")
    experts, hidden_out, hidden_in = 3, 28672, 65536   # 5.6e9 bytes
    b = torch.empty(experts, hidden_out, hidden_in, dtype=torch.int8, device="cuda").random_(-128, 128)
    sb = torch.rand(experts, hidden_out, device="cuda") / 64 + 1e-3
    for rows, sizes in ((4, [1, 1, 2]), (120, [40, 50, 30])):
        a = torch.empty(rows, hidden_in, dtype=torch.int8, device="cuda").random_(-128, 128)
        sa = torch.rand(rows, device="cuda") / 64 + 1e-3
        got = ops.gmm_int8(a, sa, b, sb, torch.tensor(sizes).cuda())
        for e, first in ((0, 0), (2, rows - 1)):
            at = slice(hidden_out - 300, hidden_out)
            want = (a[first].double() @ b[e, at].double().t() * sa[first].double() * sb[e, at].double()).cpu()
            _check_close(got[first, at], want, torch.bfloat16, (rows, e))
    del b, a, got
    rows, hidden_in = 1 << 18, 17408   # 4.6e9 bytes
    x = torch.randn(512, hidden_in, device="cuda", dtype=torch.bfloat16)
    index = (torch.arange(rows, device="cuda") % 512).to(torch.int32)
    q = ops.quantize_rows(x, index)
    want, scales = _quantized(x.cpu())
    for r in (0, 511, rows - 513, rows - 1):
        assert torch.equal(q.values[r].cpu(), want[r % 512]) and q.scales[r].cpu() == scales[r % 512], r
    b = torch.randint(-128, 128, (2, 24, hidden_in), dtype=torch.int8, device="cuda")
    sb = torch.rand(2, 24, device="cuda") + 0.5
    got = ops.gmm_int8(q.values, q.scales, b, sb, torch.tensor([rows - 1000, 1000]))
    for r in (0, rows - 1001, rows - 1000, rows - 1):
        e = 0 if r < rows - 1000 else 1
        want_r = (want[r % 512].double() @ b[e].double().cpu().t()) * scales[r % 512].double() * sb[e].double().cpu()
        _check_close(got[r], want_r, torch.bfloat16, r)


def test_an_expert_layer_in_8_bits(ops):
    """A run of the operators together, routed, against the same layer in 64 bits on the values that the 8-bit numbers stand for; quantising the rows
    in between moves each by half a step, 1/254 of its row's largest, which the next product averages over its depth."""
    _announce("layer")
    tokens, experts, k, hidden, ffn = 200, 8, 2, 256, 320
    g = torch.Generator().manual_seed(1)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16).cuda()
    w13 = ops.quantize_rows((torch.randn(experts, 2 * ffn, hidden, generator=g) * hidden ** -0.5).cuda())
    w2 = ops.quantize_rows((torch.randn(experts, hidden, ffn, generator=g) * ffn ** -0.5).cuda())
    r = ops.route(torch.randn(tokens, experts, generator=g).cuda(), k)
    q = ops.quantize_rows(x, r.row_index)
    gate_up = ops.gmm_int8(q.values, q.scales, w13.values, w13.scales, r.batch_sizes)
    h = ops.swiglu_quantize(gate_up)
    # (the router's weights go into the scales of the second product's rows)
    rows = ops.gmm_int8(h.values, h.scales * r.weights.view(-1)[r.order.long()], w2.values, w2.scales, r.batch_sizes)
    out = torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda").index_add_(0, r.row_index.long(), rows.double())
    of_row = torch.repeat_interleave(torch.arange(experts, device="cuda"), r.batch_sizes)
    real = lambda v: v.values.double() * v.scales.double().unsqueeze(-1)  # noqa: E731

    def product(w, q, scales):   # (whole numbers first, so that what cancels does)
        return torch.matmul(w.values[of_row].double(), q.values.double().unsqueeze(2)).squeeze(2) * w.scales[of_row].double() * scales.unsqueeze(1)

    both = product(w13, q, q.scales.double())
    _check_close(gate_up, both.cpu(), torch.bfloat16, "first product")
    gate, up = gate_up.double().chunk(2, 1)
    exact_h = torch.nn.functional.silu(gate) * up
    assert ((real(h) - exact_h).abs() <= 0.501 * h.scales.double().unsqueeze(1)).all()
    want = product(w2, h, h.scales.double() * r.weights.double().view(-1)[r.order.long()])
    # (a weight times a scale is rounded once more: 2^-24)
    assert ((rows.double() - want).abs() <= (2.0 ** -8 + 5 * 2.0 ** -24) * want.abs()).all()
    dense = torch.matmul(real(w2)[of_row], exact_h.unsqueeze(2)).squeeze(2) * r.weights.double().view(-1)[r.order.long()].unsqueeze(1)
    dense = torch.zeros_like(out).index_add_(0, r.row_index.long(), dense)
    assert float((out - dense).norm() / dense.norm()) < 0.02
