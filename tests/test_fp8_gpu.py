"""The block-scaled 8-bit operators against plain 64-bit implementations.

Bounds: a value rounded to 8 bits is compared bit for bit (its scale is a power of two, so there is one rounding).  A product's sum of K terms in 32 bits
is off by at most K 2^-23 of the sum of magnitudes (a unit in the last place for each addition, whatever the order), and rounding to the result's type adds half
a step, eps / 2."""
import copy
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch
import torch.utils.checkpoint

from venom_b200 import capi, fp8

pytestmark = pytest.mark.gpu
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---- plain forms in 64 bits ----

def pow2(e):
    """2^e, bit for bit, for whole numbers e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def exponent(v):
    """floor(log2 v) of positive v, without the rounding of a logarithm."""
    return (torch.frexp(v)[1] - 1).double()


def held64(x, f8=E4M3, square=False):
    """(units, exponents): values in units of their block's scale, and log2 of the scale of each row and block."""
    top, low, bits = (448.0, -6, 3) if f8 == E4M3 else (57344.0, -14, 2)
    x = x.detach().double()
    n, k = x.shape
    tall = 128 if square else 1
    nb, kb = -(-n // tall), -(-k // 128)
    full = x.new_zeros((nb * tall, kb * 128))
    full[:n, :k] = x
    b = full.view(nb, tall, kb, 128)
    amax = torch.where(b.isfinite(), b.abs(), torch.zeros_like(b)).amax(dim=(1, 3), keepdim=True)
    e = torch.where(amax > 0, exponent(amax) - exponent(torch.tensor(top, dtype=torch.float64)).item(), torch.full_like(amax, -127)).clamp(min=-127)
    e = torch.where(amax > top * pow2(e), e + 1, e)
    v = b * pow2(-e)
    step = pow2(exponent(torch.where(v.isfinite(), v.abs(), torch.ones_like(v)).clamp(min=2.0 ** low)) - bits)
    q = torch.where(v.isfinite(), torch.round(v / step) * step, v)
    return q.reshape(nb * tall, kb * 128)[:n, :k], e.expand(nb, tall, kb, 1).reshape(nb * tall, kb)[:n]


def value64(x, f8=E4M3, square=False):
    q, e = held64(x, f8, square)
    return q * pow2(e).repeat_interleave(128, 1)[:, : q.shape[1]]


def unpacked(q):
    n, k = q.shape
    e = q.scales.view(torch.uint8).permute(1, 0, 2).reshape(n, -1)[:, : -(-k // 128)].double() - 127
    return q.data.double(), e


def check_held(q, x, f8, square=False):
    want, we = held64(x, f8, square)
    got, ge = unpacked(q)
    assert torch.equal(ge, we), "scales"
    if f8 == E4M3:
        want = torch.where(want.isinf(), torch.full_like(want, math.nan), want)
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9)), "values"
    blocks = -(-x.shape[1] // 128)
    assert int(q.scales.view(torch.uint8).permute(1, 0, 2).reshape(x.shape[0], -1)[:, blocks:].sum()) == 0, "bytes past the last block"


def check_product(got, a, b, bias=None, what=""):
    """got against a @ b.T + bias of 64-bit matrices."""
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps       # a step of denormal results
    bound = (a.shape[1] + 1) * 2.0 ** -23 * size * (1 + eps) + eps * want.abs() + tiny
    far = (got.double() - want).abs() - bound
    assert got.shape == want.shape and not bool((far > 0).any()), "%s: %g over the bound" % (what, far.max().item())


def matrix(rows, cols, seed, dtype=torch.float32, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, cols), device="cuda", generator=g)
    return (x * torch.exp(spread * torch.randn((rows, 1), device="cuda", generator=g))).to(dtype)


def vector(n, seed, dtype):
    return matrix(1, n, seed, dtype, 0.0)[0]


# ---- quantise ----

@pytest.mark.parametrize("f8", [E4M3, E5M2])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (2, 129), (7, 8), (128, 128), (129, 511), (130, 513), (1000, 17), (5, 4099), (333, 1032)])
def test_quantize(rows, cols, dtype, square, f8):
    x = matrix(rows, cols, rows + cols, TYPES[dtype], 2.0)
    q, t = fp8.quantize(x, f8, square=square, both=True)
    check_held(q, x, f8, square)
    check_held(t, x.t(), f8, square)
    check_held(fp8.quantize(x, f8, square=square), x, f8, square)
    for dt in TYPES.values():
        want = value64(x, f8, square).to(torch.float32).to(dt)      # exact in 32 bits
        assert torch.equal(q.dequantize(dt), want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("f8", [E4M3, E5M2])
def test_quantize_extremes(dtype, square, f8):
    t = TYPES[dtype]
    info = torch.finfo(t)
    x = matrix(260, 700, 3, t)
    x[0] = 0                                          # nothing in the row
    x[1, :128], x[1, 128:256] = info.max, -info.max    # the lowest value, as masks use it
    x[2, 5], x[2, 200], x[2, 400] = math.nan, math.inf, -math.inf
    x[3] = math.inf                                   # no finite value in the row
    x[4] = info.smallest_normal * info.eps            # the smallest denormal
    x[5], x[5, 0] = info.smallest_normal, info.max    # values far below the block's scale
    x[6:8, 128] = torch.tensor([1.75, 1.7500001 if dtype == "fp32" else 1.75 + 2 * info.eps], device="cuda").to(t)
    x[6:8, 129:256] = 0.5                              # either side of the line between two scales
    x[:, 300] = math.nan
    x[:, 301] = 0
    q, tr = fp8.quantize(x, f8, square=square, both=True)
    check_held(q, x, f8, square)
    check_held(tr, x.t(), f8, square)
    check_held(fp8.quantize(x, f8, square=square), x, f8, square)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize_reads_strided_and_unaligned_rows(dtype):
    base = matrix(70, 401, 9, TYPES[dtype])
    for x in (base[:, 1:], base[:, 3:259], base[5:6, :130], base.t(), base[::2, :], base[:, ::3], base[1:, 8:264], base[:1].expand(70, 401)):
        q, t = fp8.quantize(x, both=True)
        check_held(q, x, E4M3)
        check_held(t, x.t(), E4M3)
        check_held(fp8.quantize(x), x, E4M3)


@pytest.mark.parametrize("rows,cols", [(5, 130), (130, 5), (257, 260)])
def test_quantize_writes_its_own_rows_only(rows, cols):
    """Through the C ABI: what lies behind the rows, and between them past the padding that the call owns, stays."""
    x = matrix(rows, cols, 1, torch.float16)
    ld, ldt = -(-cols // 16) * 16 + 32, -(-rows // 16) * 16 + 32
    data, data_t = (torch.full((n + 2, d), 0xA5, dtype=torch.uint8, device="cuda") for n, d in ((rows, ld), (cols, ldt)))
    lib = capi.lib()
    sizes = [lib.vnm_fp8_scale_bytes(rows, cols), lib.vnm_fp8_scale_bytes(cols, rows)]
    s, st = (torch.full((n + 64,), 0xA5, dtype=torch.uint8, device="cuda") for n in sizes)
    ws, sums = torch.full((-(-rows // 128) * cols + 16,), 7.0, device="cuda"), torch.full((cols + 16,), 7.0, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.vnm_fp8_quantize(x.data_ptr(), 1, cols, rows, cols, 0, 0, data.data_ptr(), ld, s.data_ptr(), data_t.data_ptr(), ldt, st.data_ptr(), sums.data_ptr(), 0, ws.data_ptr(),
                                stream) == 0
    for d, n, k in ((data, rows, cols), (data_t, cols, rows)):
        assert bool((d[n:] == 0xA5).all()) and bool((d[:, -(-k // 16) * 16:] == 0xA5).all())
        assert int((d[:n, k:-(-k // 8) * 8] != 0).sum()) == 0
    assert bool((s[sizes[0]:] == 0xA5).all()) and bool((st[sizes[1]:] == 0xA5).all())
    assert bool((ws[-(-rows // 128) * cols:] == 7).all()) and bool((sums[cols:] == 7).all())
    want = x.double().sum(0)
    assert bool(((sums[:cols].double() - want).abs() <= rows * 2.0 ** -23 * x.double().abs().sum(0)).all())
    check_held(fp8.BlockFp8(data[:rows, :cols].view(E4M3), s[: sizes[0]].view(-1, rows, 4).view(torch.float8_e8m0fnu)), x, E4M3)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", [1, 5, 7, 8, 9, 15, 17, 120, 127, 129, 505, 511, 513, 1031])
def test_rows_that_begin_anywhere(dtype, cols):
    """Every offset of a row inside 16 bytes, for what is read (values) and written (GELU and its gradient), and nothing written beside the rows."""
    t = TYPES[dtype]
    for start in range(0, 16 // t.itemsize):
        x = matrix(11, cols, cols + start, t)
        base = torch.zeros(11 * cols + 64, dtype=t, device="cuda")
        moved = base[start:start + 11 * cols].view(11, cols)
        moved.copy_(x)
        base[:start], base[start + 11 * cols:] = math.nan, math.inf            # neighbours that must not get in
        for both in (False, True):
            q = fp8.quantize(moved, both=both)
            check_held(q[0] if both else q, x, E4M3)
            if both:
                check_held(q[1], x.t(), E4M3)
        lib, stream, tcode = capi.lib(), torch.cuda.current_stream().cuda_stream, {"fp32": 0, "fp16": 1, "bf16": 2}[dtype]
        h = fp8.quantize(x)
        y = torch.full((11 * cols + 64,), 7.0, dtype=t, device="cuda")
        at = y.data_ptr() + start * t.itemsize
        assert lib.vnm_fp8_gelu(moved.data_ptr(), tcode, cols, 11, cols, 0, at, cols, None, 16, None, None, 16, None, None, 16, None, stream) == 0
        check_gelu(y[start:start + 11 * cols].view(11, cols), gelu64(x, False)[0], x)
        assert bool((y[:start] == 7).all()) and bool((y[start + 11 * cols:] == 7).all())
        y.fill_(7.0)
        assert lib.vnm_fp8_gelu_grad(moved.data_ptr(), tcode, cols, 11, cols, 1, h.data.data_ptr(), h.data.stride(0), h.scales.data_ptr(), at, cols, 0, None, 16, None, None, 16, None,
                                     None, 0, None, stream) == 0
        check_gelu(y[start:start + 11 * cols].view(11, cols), x.double() * gelu64(value64(x), True)[1], value64(x), x)
        assert bool((y[:start] == 7).all()) and bool((y[start + 11 * cols:] == 7).all())


@pytest.mark.parametrize("f8", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 9), (257, 511), (128, 512), (1000, 130), (2, 4099)])
def test_dequantize(rows, cols, dtype, f8):
    """Every value is exact in 32 bits, so it is rounded once; rows of the result may begin anywhere."""
    x, t = matrix(rows, cols, 5), TYPES[dtype]
    x[0, 0] = float("nan")
    q = fp8.quantize(x, f8)
    want = value64(x, f8).float().to(t)
    same = lambda got: bool(((got == want) | (got.isnan() & want.isnan())).all())
    assert q.dequantize(t).dtype == t and same(q.dequantize(t))
    code, lib = {"fp16": 1, "bf16": 2, "fp32": 0}[dtype], capi.lib()
    for shift, ldo in ((1, cols + 3), (2, cols + 6), (0, cols + 8)):
        base = torch.full((rows * ldo + 8,), 7.0, dtype=t, device="cuda")
        assert lib.vnm_fp8_dequantize(q.data.data_ptr(), q.data.stride(0), q.scales.data_ptr(), 0 if f8 == E4M3 else 1, rows, cols, base[shift:].data_ptr(), code, ldo,
                                      torch.cuda.current_stream().cuda_stream) == 0
        out = base[shift: shift + rows * ldo].view(rows, ldo)
        assert same(out[:, :cols]) and bool((base[:shift] == 7).all()) and bool((out[:, cols:] == 7).all()) and bool((base[shift + rows * ldo:] == 7).all())


def test_quantize_long_rows_and_many_rows():
    """Offsets past 32 bits in the input and the result."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    rows, cols = 70000, 65600                        # 4.6 G values
    x = torch.zeros((rows, cols), dtype=torch.float16, device="cuda")
    x[-3:] = matrix(3, cols, 2, torch.float16)
    x[0] = matrix(1, cols, 4, torch.float16)[0]
    x[:, -2] = 3.0
    q = fp8.quantize(x)
    for at in (0, rows - 3, rows - 1):
        check_held(fp8.BlockFp8(q.data[at:at + 1], q.scales[:, at:at + 1].contiguous()), x[at:at + 1], E4M3)
    del q
    _, t = fp8.quantize(x, both=True)
    for at in (0, cols - 2, cols - 1):
        check_held(fp8.BlockFp8(t.data[at:at + 1], t.scales[:, at:at + 1].contiguous()), x[:, at:at + 1].t(), E4M3)


# ---- products ----

SHAPES = [(1, 1, 1), (1, 8, 16), (8, 1024, 1024), (16, 136, 512), (17, 128, 640), (33, 1000, 1024), (64, 300, 130), (65, 257, 127), (128, 128, 128), (129, 129, 1537),
          (256, 512, 2048), (300, 700, 2039), (511, 1030, 777), (1000, 40, 4096), (40, 1000, 4096), (1024, 2048, 256), (2049, 515, 384)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("types", [(E4M3, E4M3, "fp16"), (E5M2, E4M3, "bf16"), (E4M3, E5M2, "fp32")])
@pytest.mark.parametrize("bias", [None, "fp16", "fp32"])
def test_matmul(M, N, K, types, bias):
    a, b = fp8.quantize(matrix(M, K, M + K), types[0]), fp8.quantize(matrix(N, K, N + K + 1, spread=0.3), types[1], square=True)
    bias = None if bias is None else vector(N, 5, TYPES[bias])
    got = fp8.matmul(a, b, bias, TYPES[types[2]])
    check_product(got, value64(a.dequantize().double(), types[0]), value64(b.dequantize().double(), types[1]), bias)
    assert torch.equal(got, fp8.matmul(a, b, bias, TYPES[types[2]])), "two calls differ"
    assert fp8.device_status() == 0


# (columns of a pair tile, rows in whole pieces, at least two tiles for every pair of SMs, 32-bit results, bias): a shape that takes that instance
INSTANCES = {
    (192, False, False, False, False): (5054, 129, 628), (192, False, False, True, False): (4787, 135, 626), (192, False, True, False, False): (2324, 3678, 602),
    (192, False, True, True, False): (5406, 1562, 611), (192, True, False, False, False): (2656, 136, 730), (192, True, False, True, True): (2651, 140, 640),
    (192, True, True, False, False): (2361, 3632, 628), (192, True, True, True, True): (1555, 5552, 619), (224, False, False, False, True): (525, 4729, 652),
    (224, False, False, True, True): (521, 4630, 615), (224, False, True, False, False): (1580, 5980, 610), (224, False, True, True, True): (2049, 4681, 604),
    (224, True, False, False, False): (524, 4968, 644), (224, True, False, True, True): (559, 4964, 614), (224, True, True, False, True): (1797, 5424, 615),
    (224, True, True, True, True): (1794, 5396, 601), (240, False, False, False, False): (4657, 674, 605), (240, False, False, True, False): (576, 5386, 620),
    (240, False, True, False, True): (3358, 3439, 602), (240, False, True, True, True): (2060, 5487, 600), (240, True, False, False, False): (519, 5680, 632),
    (240, True, False, True, True): (563, 5508, 613), (240, True, True, False, False): (2909, 4072, 619), (240, True, True, True, True): (2113, 5428, 604),
    (256, False, False, False, False): (513, 5783, 660), (256, False, False, True, True): (544, 5938, 622), (256, False, True, False, True): (2561, 4993, 670),
    (256, False, True, True, True): (2305, 5609, 711), (256, True, False, False, False): (807, 4472, 630), (256, True, False, True, False): (542, 5996, 645),
    (256, True, True, False, False): (2306, 5576, 603), (256, True, True, True, True): (2563, 5000, 710)}


def plan_of(M, N, K, dtype, bias):
    v = [ctypes.c_int() for _ in range(4)]
    whole = N * torch.finfo(dtype).bits // 8 % 16 == 0     # rows of a contiguous result
    assert capi.lib().vnm_fp8_matmul_config(M, N, K, 0 if dtype == torch.float32 else 1, whole, bias, *[ctypes.byref(x) for x in v]) == 0
    return [x.value for x in v]


@pytest.mark.parametrize("instance", list(INSTANCES), ids=lambda i: "-".join(map(str, i)))
def test_matmul_pair_instances(instance):
    width, _, _, wide, with_bias = instance
    M, N, K = INSTANCES[instance]
    for dtype in (torch.float32,) if wide else (torch.float16, torch.bfloat16):
        assert plan_of(M, N, K, dtype, with_bias)[:2] == [256, width]
        a, b = fp8.quantize(matrix(M, K, M, spread=0.5)), fp8.quantize(matrix(N, K, N, spread=0.3), E5M2)
        bias = vector(N, 5, dtype) if with_bias else None
        got = fp8.matmul(a, b, bias, dtype)
        check_product(got, a.dequantize().double(), b.dequantize().double(), bias)
        assert torch.equal(got, fp8.matmul(a, b, bias, dtype)), "two calls differ"
    assert fp8.device_status() == 0


@pytest.mark.parametrize("M,N,K,want", [(62, 10, 25, (16, 1)), (623, 8, 1252, (16, 2)), (1, 855, 720, (16, 4)), (1, 115, 1123, (16, 8)), (2496, 171, 16, (32, 1)), (1631, 8, 2666, (32, 2)),
                                        (762, 9, 4578, (32, 4)), (399, 11, 6782, (32, 8)), (513, 1877, 7239, (64, 1)), (102, 2313, 3731, (64, 2)), (1857, 8, 6344, (64, 4)), (40, 2195, 7979, (64, 8)),
                                        (3125, 239, 7948, (128, 4))])
def test_matmul_one_sm_instances(M, N, K, want):
    dtype = torch.float32 if want[0] == 128 else torch.float16
    tile_m, tile_n, split, _ = plan_of(M, N, K, dtype, False)
    assert (tile_m, split) == want and tile_n == 128
    a, b = fp8.quantize(matrix(M, K, M, spread=0.5)), fp8.quantize(matrix(N, K, N, spread=0.3), E5M2)
    check_product(fp8.matmul(a, b, None, dtype), a.dequantize().double(), b.dequantize().double())
    assert fp8.device_status() == 0


@pytest.mark.parametrize("M,N,K,dtype", [(70000, 40008, 136, torch.float16), (40007, 33001, 40, torch.float32)])
def test_matmul_results_past_32_bits(M, N, K, dtype):
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    a, b = fp8.quantize(matrix(M, K, 1, spread=0.3)), fp8.quantize(matrix(N, K, 2, spread=0.3))
    got = fp8.matmul(a, b, None, dtype)
    rows = torch.tensor([0, 1, 255, 256, M // 2, M - 257, M - 2, M - 1], device="cuda")
    check_product(got[rows], a.dequantize()[rows].double(), b.dequantize().double())


def test_matmul_operands_past_32_bits():
    """A weight of 4.4 GB."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    N, K = 70000, 62992
    data = torch.zeros((N, K), dtype=torch.uint8, device="cuda")
    scales = torch.full((-(-K // 512), N, 4), 127, dtype=torch.uint8, device="cuda")
    last = matrix(300, K, 3, spread=0.3)
    q = fp8.quantize(last)
    data[-300:] = q.data.view(torch.uint8)
    scales[:, -300:] = q.scales.view(torch.uint8)
    x = fp8.quantize(matrix(5, K, 4))
    got = fp8.matmul(x, fp8.BlockFp8(data.view(E4M3), scales.view(torch.float8_e8m0fnu)), dtype=torch.float32)
    assert bool((got[:, :-300] == 0).all())
    check_product(got[:, -300:], x.dequantize().double(), q.dequantize().double())


def test_matmul_scales_of_every_size():
    """Rows and blocks whose scales lie far apart, blocks of nothing, and rows of nothing."""
    x = matrix(200, 1500, 1)
    x *= torch.exp2(torch.randint(-20, 20, (200, 1), device="cuda").float())
    x[:, 128:256] *= 2.0 ** -10
    x[3] = 0
    x[5, 256:512] = 0
    w = matrix(140, 1500, 2)
    w[:, 700:] *= 2.0 ** 12
    a, b = fp8.quantize(x), fp8.quantize(w)
    got = fp8.matmul(a, b, dtype=torch.float32)
    check_product(got, value64(x), value64(w))
    assert bool((got[3] == 0).all())


def test_matmul_values_that_are_not_finite():
    x, w = matrix(40, 300, 1), matrix(130, 300, 2)
    x[7, 290] = math.nan
    w[9, 3] = math.inf
    got = fp8.matmul(fp8.quantize(x), fp8.quantize(w), dtype=torch.float32)
    bad = torch.zeros((40, 130), dtype=torch.bool, device="cuda")
    bad[7], bad[:, 9] = True, True
    assert torch.equal(got.isnan(), bad)


def test_matmul_reads_operands_as_they_lie():
    """Rows further apart than they are long, and what lies past the last column or row is not read."""
    M, N, K = 70, 150, 300
    x, w = matrix(M, K, 1), matrix(N, K, 2)
    a, b = fp8.quantize(x), fp8.quantize(w)
    big = torch.full((M + 4, 448), 0x7F, dtype=torch.uint8, device="cuda")               # NaN all around
    big[2:2 + M, 16:16 + K] = a.data.view(torch.uint8)
    view = big.view(E4M3)[2:2 + M, 16:16 + K]
    assert torch.equal(fp8.matmul(fp8.BlockFp8(view, a.scales), b), fp8.matmul(a, b))
    assert torch.equal(fp8.matmul(b, fp8.BlockFp8(view, a.scales)), fp8.matmul(b, a))
    with pytest.raises(capi.VenomError, match="16"):
        fp8.matmul(fp8.BlockFp8(big.view(E4M3)[2:2 + M, 17:17 + K], a.scales), b)


@pytest.mark.parametrize("M,N,ldo", [(33, 130, 161), (300, 257, 300), (5, 64, 64), (257, 520, 528), (2051, 1999, 2000), (2050, 1999, 2008), (2050, 1993, 1999), (1500, 2053, 2056)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_matmul_writes_its_own_rows_only(M, N, ldo, dtype):
    K = 520
    a, b = fp8.quantize(matrix(M, K, 1)), fp8.quantize(matrix(N, K, 2))
    out = torch.full((M + 2, ldo), 7.0, dtype=TYPES[dtype], device="cuda")
    assert capi.lib().vnm_fp8_matmul(a.data.data_ptr(), a.data.stride(0), a.scales.data_ptr(), 0, b.data.data_ptr(), b.data.stride(0), b.scales.data_ptr(), 0, M, N, K, None, 0,
                                     out.data_ptr(), {"fp32": 0, "fp16": 1, "bf16": 2}[dtype], ldo, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out[:M, :N], fp8.matmul(a, b, dtype=TYPES[dtype]))
    assert bool((out[M:] == 7).all()) and bool((out[:, N:] == 7).all())


def test_matmul_refusals():
    a, b = fp8.quantize(matrix(8, 256, 1)), fp8.quantize(matrix(16, 256, 2))
    for call, match in ((lambda: fp8.matmul(a, fp8.quantize(matrix(16, 128, 2))), "do not match"), (lambda: fp8.matmul(a, b, vector(15, 1, torch.float16)), "bias"),
                        (lambda: fp8.matmul(a, b, dtype=torch.float64), "fp32 expected"), (lambda: fp8.matmul(fp8.BlockFp8(a.data, b.scales), b), "scales"),
                        (lambda: fp8.matmul(fp8.BlockFp8(a.data, a.scales.cpu()), b), "CUDA device"), (lambda: fp8.matmul(a, b, vector(16, 1, torch.float16).cpu()), "bias"),
                        (lambda: fp8.quantize(matrix(8, 8, 1).double()), "fp32 expected"), (lambda: fp8.quantize(matrix(8, 8, 1), torch.float16), "float8"),
                        (lambda: fp8.quantize(matrix(8, 8, 1)[0]), "matrix")):
        with pytest.raises(capi.VenomError, match=match):
            call()


def test_empty_operands():
    x = matrix(0, 300, 1, torch.float16)
    q, t = fp8.quantize(x, both=True)
    assert q.shape == (0, 300) and t.shape == (300, 0)
    b = fp8.quantize(matrix(16, 300, 1))
    assert fp8.matmul(q, b).shape == (0, 16) and fp8.matmul(b, q).shape == (16, 0)
    assert q.dequantize().shape == (0, 300)


# ---- linear ----

def leaf(t):
    return t.detach().clone().requires_grad_()


@pytest.mark.parametrize("shape,cin,cout", [((1,), 64, 64), ((37,), 200, 131), ((2, 5, 3), 129, 257), ((128,), 128, 128), ((600,), 1000, 520), ((0,), 64, 32), ((2, 0), 64, 32)])
@pytest.mark.parametrize("x_type,w_type,grad_dtype", [("fp16", "fp16", E4M3), ("bf16", "fp32", E4M3), ("fp32", "bf16", E5M2)])
def test_linear(shape, cin, cout, x_type, w_type, grad_dtype):
    tokens = math.prod(shape)
    x = leaf(matrix(tokens, cin, 1, TYPES[x_type]).reshape(*shape, cin))
    w, b = leaf(matrix(cout, cin, 2, TYPES[w_type], 0.2)), leaf(vector(cout, 3, TYPES[w_type]))
    dy = matrix(tokens, cout, 4, TYPES[x_type]).reshape(*shape, cout)
    y = fp8.linear(x, w, b, grad_dtype)
    assert y.shape == dy.shape and y.dtype == x.dtype
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (dx.shape, dx.dtype, dw.shape, dw.dtype, db.shape, db.dtype) == (x.shape, x.dtype, w.shape, w.dtype, b.shape, b.dtype)
    if tokens == 0:
        assert bool((dw == 0).all()) and bool((db == 0).all())
        return
    x2, dy2 = x.detach().reshape(tokens, cin), dy.reshape(tokens, cout)
    hw = value64(w, square=True)
    check_product(y.detach().reshape(tokens, cout), value64(x2), hw, b.detach(), "y")
    check_product(dx.reshape(tokens, cin), value64(dy2, grad_dtype), hw.t(), None, "dx")
    check_product(dw, value64(dy2.t(), grad_dtype), value64(x2.t()), None, "dw")
    check_product(db[None], torch.ones((1, tokens), dtype=torch.float64, device="cuda"), dy2.double().t(), None, "db")
    # the gradient of the layer without its roundings: each 8-bit factor is off by half a step of its type, 2^-4 for e4m3 and 2^-3 for e5m2 (and by half
    # of the smallest step where a value is far below its block's scale: 2^-10 of amax / 224 or 2^-17 of amax / 28672)
    rel = (1 + 2.0 ** -4) * (1 + (2.0 ** -4 if grad_dtype == E4M3 else 2.0 ** -3)) - 1
    exact = dy2.double() @ w.detach().double()
    size = dy2.double().abs() @ w.detach().double().abs()
    floor = cout * 2.0 ** -17 * dy2.double().abs().amax(1, keepdim=True) * w.detach().double().abs().amax()
    assert bool(((dx.reshape(tokens, cin).double() - exact).abs() <= rel * size + 2 * floor + torch.finfo(dx.dtype).eps * size + 1e-7).all())


def test_linear_gives_only_the_gradients_that_are_wanted():
    x, w, b, dy = matrix(40, 200, 1, torch.float16), matrix(72, 200, 2, torch.float16), vector(72, 3, torch.float16), matrix(40, 72, 4, torch.float16)
    leaves = [leaf(x), leaf(w), leaf(b)]
    full = torch.autograd.grad(fp8.linear(*leaves), leaves, dy)
    for mask in range(1, 8):
        some = [leaf(t) if mask >> i & 1 else t for i, t in enumerate((x, w, b))]
        y = fp8.linear(*some)
        y.backward(dy)
        for i in range(3):
            assert (some[i].grad is None) if not mask >> i & 1 else torch.equal(some[i].grad, full[i])
    assert not fp8.linear(x, w, b).requires_grad
    with torch.no_grad():
        assert torch.equal(fp8.linear(*leaves), fp8.linear(x, w, b))


def test_linear_shared_weight_and_strided_gradients():
    """One weight used twice; gradients that arrive broadcast or transposed."""
    x, w = leaf(matrix(50, 96, 1, torch.bfloat16)), leaf(matrix(96, 96, 2, torch.bfloat16))
    (fp8.linear(x, w) + fp8.linear(x, w)).sum().backward()
    g1 = torch.autograd.grad(fp8.linear(x, w), (x, w), torch.ones((50, 96), dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(w.grad, g1[1] + g1[1]) and torch.equal(x.grad, g1[0] + g1[0])
    dy = matrix(96, 50, 5, torch.bfloat16)
    a, b = torch.autograd.grad(fp8.linear(x, w), w, dy.t())[0], torch.autograd.grad(fp8.linear(x, w), w, dy.t().contiguous())[0]
    assert torch.equal(a, b)


def test_linear_refusals():
    x, w = matrix(4, 64, 1, torch.float16), matrix(8, 64, 2, torch.float16)
    for call, match in ((lambda: fp8.linear(x[:, :32], w), "do not match"), (lambda: fp8.linear(x, w, vector(7, 1, torch.float16)), "bias"), (lambda: fp8.linear(x.double(), w), "expected"),
                        (lambda: fp8.linear(x, w.cpu()), "device"), (lambda: fp8.linear(x, w, grad_dtype=torch.float16), "gradients"), (lambda: fp8.linear(x.long(), w), "expected"),
                        (lambda: fp8.gelu(x, "fast"), "approximate"), (lambda: fp8.mlp(x, w, None, w, None), "do not match")):
        with pytest.raises(capi.VenomError, match=match):
            call()
    y = fp8.linear(leaf(x), leaf(w))
    (g,) = torch.autograd.grad(y.float().square().sum(), y, create_graph=True)
    xl = leaf(x)
    y = fp8.linear(xl, w)
    (g,) = torch.autograd.grad(y.float().square().sum(), xl, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), xl)


# ---- GELU ----

def gelu64(x, tanh):
    x = x.double()
    if tanh:
        u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        s = torch.sigmoid(2 * u)
        return x * s, s + x * s * torch.sigmoid(-2 * u) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * x ** 2)
    cdf = torch.special.ndtr(x)
    return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


# The approximation of erfc is off by 1.5e-7, so Phi by 0.75e-7; its polynomial, the exponential and the reciprocal add at most ten roundings of 2^-24 to values up
# to 1 (the exponent's argument, x^2 / 2 log2 e <= 150 where the result is not zero, is rounded too: 150 2^-24 ln 2 of a density that is then below 2^-100,
# at most 2^-24 of x times the density for any x).  2e-6 (1 + |x|) covers both; the tanh form has fewer.
def check_gelu(got, want, x, scale=None, extra=0.0):
    scale = torch.ones_like(want) if scale is None else scale.double().abs()
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    far = (got.double() - want).abs() - (2e-6 * (1 + x.double().abs()) * scale + eps * want.abs() + tiny)
    assert not bool((far > 0).any()), far.max().item()


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 130), (128, 128), (257, 777), (64, 4096), (0, 64)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tanh", [False, True])
def test_gelu(rows, cols, dtype, tanh):
    x, dy = leaf(matrix(rows, cols, 1, TYPES[dtype])), matrix(rows, cols, 2, TYPES[dtype])
    y = fp8.gelu(x, "tanh" if tanh else "none")
    (dx,) = torch.autograd.grad(y, x, dy)
    h = value64(x) if rows else x.detach().double()
    check_gelu(y.detach(), gelu64(x.detach(), tanh)[0], x.detach())
    check_gelu(dx, dy.double() * gelu64(h, tanh)[1], h, dy)
    if rows:   # against differences of the function at what the checkpoint holds: a central difference of step d is off by at most d^2 / 6 of a third derivative below 2
        d = 1e-5
        slope = (gelu64(h + d, tanh)[0] - gelu64(h - d, tanh)[0]) / (2 * d)
        check_gelu(dx, dy.double() * slope, h, dy)
    with torch.no_grad():
        assert torch.equal(fp8.gelu(x, "tanh" if tanh else "none"), y)


@pytest.mark.parametrize("tanh", [False, True])
def test_gelu_far_values(tanh):
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 6.0, -6.0, 13.0, -13.0, 100.0, -100.0, 3e4, -3e4, 1e30, -1e30, 3e38, -3e38], device="cuda")
    x = leaf(v[:, None].expand(16, 4).contiguous())          # a block each: the checkpoint holds the values themselves
    y = fp8.gelu(x, "tanh" if tanh else "none")
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    big = v.abs() > 20
    assert torch.equal(y[big], torch.where(v > 0, v, torch.zeros_like(v))[big][:, None].expand(-1, 4))
    assert torch.equal(dx[big], (v > 0).float()[big][:, None].expand(-1, 4))
    check_gelu(y[~big].detach(), gelu64(x.detach()[~big], tanh)[0], x.detach()[~big])
    x = matrix(4, 200, 1)
    x[1, 3], x[2, 150] = math.nan, math.inf
    x = leaf(x)
    y = fp8.gelu(x, "tanh" if tanh else "none")
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(y.isnan(), x.isnan()) and bool(y[2, 150].isinf())
    assert torch.equal(dx.isnan(), x.isnan() | x.isinf())     # e4m3 holds an infinity as NaN


def test_gelu_of_any_shape_and_strides():
    x = leaf(matrix(60, 210, 1, torch.float16))
    dy = matrix(60, 210, 2, torch.float16)
    want = fp8.gelu(x)
    (dw,) = torch.autograd.grad(want, x, dy)
    y = fp8.gelu(x.reshape(3, 4, 5, 210))
    (dx,) = torch.autograd.grad(y, x, dy.reshape(3, 4, 5, 210))
    assert torch.equal(y.reshape(60, 210), want) and torch.equal(dx, dw)
    xt = leaf(x.detach().t().contiguous())
    y = fp8.gelu(xt.t())
    (dx,) = torch.autograd.grad(y, xt, dy)
    assert torch.equal(y, want) and torch.equal(dx, dw.t())
    (dx,) = torch.autograd.grad(fp8.gelu(x[:, 1:]), x, dy[:, 1:])
    assert bool((dx[:, 0] == 0).all())


# ---- feed-forward block ----

def mlp64(x, w1, b1, w2, b2, dy, tanh, t, grad_dtype):
    h1, h2 = value64(w1, square=True), value64(w2, square=True)
    h = (value64(x) @ h1.t() + b1.detach().double()).to(t).double()
    act = gelu64(h, tanh)[0]
    y = value64(act) @ h2.t() + b2.detach().double()
    dh = (value64(dy, grad_dtype) @ h2).to(t).double() * gelu64(value64(h), tanh)[1]
    return {"y": y, "dx": value64(dh, grad_dtype) @ h1, "dw1": value64(dh.t(), grad_dtype) @ value64(x.t()).t(), "db1": dh.sum(0), "dw2": value64(dy.t(), grad_dtype) @ value64(act.t()).t(),
            "db2": dy.double().sum(0)}


def block(tokens, cin, hidden, cout, t, seed=0):
    return [leaf(matrix(tokens, cin, seed + 1, t, 0.5)), leaf(matrix(hidden, cin, seed + 2, t, 0.0) * cin ** -0.5), leaf(vector(hidden, seed + 3, t)),
            leaf(matrix(cout, hidden, seed + 4, t, 0.0) * hidden ** -0.5), leaf(vector(cout, seed + 5, t))]


@pytest.mark.parametrize("tokens,cin,hidden,cout", [(1, 64, 128, 64), (70, 200, 515, 130), (300, 256, 1024, 256)])
@pytest.mark.parametrize("dtype,tanh,grad_dtype", [("fp16", False, E4M3), ("bf16", True, E4M3), ("fp32", False, E5M2)])
def test_mlp(tokens, cin, hidden, cout, dtype, tanh, grad_dtype):
    """What is kept between the halves is rounded to the type of x and then to 8 bits.  Sums that differ in their last bits may round to neighbours in that type (a
    step of eps), and of those that do a share of eps / 2^-4 lies next to a border between 8-bit values, 2^-3 apart at most: off by
    2^-3 sqrt(eps 2^4) = 2^-4.5 in the norm for bf16 (eps 2^-7) if every value did so.  A tenth of them at most do (their sums would have to be off by a tenth of a
    step, and are off by 2^-23 of their terms' size), which leaves 2^-6.  e5m2 (steps of 2^-2, with 2^3 eps): the same bound holds for fp32."""
    t = TYPES[dtype]
    leaves = block(tokens, cin, hidden, cout, t)
    dy = matrix(tokens, cout, 9, t, 0.3)
    y = fp8.mlp(*leaves, approximate="tanh" if tanh else "none", grad_dtype=grad_dtype)
    got = dict(zip(("dx", "dw1", "db1", "dw2", "db2"), torch.autograd.grad(y, leaves, dy)), y=y.detach())
    want = mlp64(*leaves, dy, tanh, t, grad_dtype)
    for k, w in want.items():
        assert got[k].shape == w.shape and got[k].dtype == t
        assert (got[k].double() - w).norm() <= 2.0 ** -6 * w.norm(), k
    with torch.no_grad():
        assert torch.equal(fp8.mlp(*leaves, approximate="tanh" if tanh else "none"), y)


def test_mlp_gives_only_the_gradients_that_are_wanted():
    values = [t.detach() for t in block(50, 96, 200, 72, torch.float16)]
    dy = matrix(50, 72, 9, torch.float16)
    leaves = [leaf(t) for t in values]
    full = torch.autograd.grad(fp8.mlp(*leaves), leaves, dy)
    for mask in range(1, 32):
        some = [leaf(t) if mask >> i & 1 else t for i, t in enumerate(values)]
        fp8.mlp(*some).backward(dy)
        for i in range(5):
            assert (some[i].grad is None) if not mask >> i & 1 else torch.equal(some[i].grad, full[i]), (mask, i)


@pytest.mark.parametrize("first,second", [(True, False), (False, True), (False, False)])
def test_mlp_with_some_biases(first, second):
    values = [t.detach() for t in block(50, 96, 200, 72, torch.float16)]
    dy = matrix(50, 72, 9, torch.float16)
    zero = [leaf(t) for t in values]
    for i, there in ((2, first), (4, second)):
        if not there:
            zero[i].data.zero_()
    want = torch.autograd.grad(fp8.mlp(*zero), zero, dy)
    for mask in range(1, 8):
        some = [leaf(t) if i in (2, 4) or mask >> (i if i < 2 else 2) & 1 else t for i, t in enumerate(values)]
        if not first:
            some[2] = None
        if not second:
            some[4] = None
        fp8.mlp(*some).backward(dy)
        for i in range(5):
            if some[i] is not None and some[i].requires_grad:
                assert torch.equal(some[i].grad, want[i]), (mask, i)


def test_mlp_without_biases_and_tokens():
    x, w1, b1, w2, b2 = block(0, 64, 128, 64, torch.float16)
    y = fp8.mlp(x, w1, None, w2, None)
    grads = torch.autograd.grad(y, (x, w1, w2), torch.empty_like(y))
    assert y.shape == (0, 64) and grads[0].shape == (0, 64) and bool((grads[1] == 0).all()) and bool((grads[2] == 0).all())


def test_gradients_without_any_output():
    """A weight without rows: nothing to sum, so the gradients behind it are zeros."""
    x, w, b = leaf(matrix(5, 64, 1, torch.float16)), leaf(torch.empty(0, 64, dtype=torch.float16, device="cuda")), leaf(torch.empty(0, dtype=torch.float16, device="cuda"))
    y = fp8.linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (5, 0) and dx.shape == x.shape and not dx.any() and dw.shape == (0, 64) and db.shape == (0,)
    w1 = leaf(matrix(96, 64, 2, torch.float16))
    y = fp8.mlp(x, w1, None, leaf(torch.empty(0, 96, dtype=torch.float16, device="cuda")), None)
    grads = torch.autograd.grad(y, (x, w1), torch.empty_like(y))
    assert y.shape == (5, 0) and not any(g.any() for g in grads)


def offloaded():
    """Saved tensors go to the host and come back."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda())


@pytest.mark.parametrize("tokens,cin,hidden,cout", [(1, 64, 128, 64), (37, 100, 203, 70), (130, 256, 512, 128)])
def test_saved_tensors_that_went_elsewhere(tokens, cin, hidden, cout):
    leaves = block(tokens, cin, hidden, cout, torch.float16)
    x, w1, b1 = leaves[:3]
    calls = ((lambda: fp8.linear(x, w1, b1), (x, w1, b1)), (lambda: fp8.gelu(x), (x,)), (lambda: fp8.mlp(*leaves), leaves))
    for call, of in calls:
        y = call()
        dy = matrix(*y.shape, 9, torch.float16)
        want = torch.autograd.grad(y, of, dy)
        with offloaded():
            y = call()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, of, dy), want))
        for reentrant in (False, True):
            y = torch.utils.checkpoint.checkpoint(lambda *_: call(), *of, use_reentrant=reentrant)
            if reentrant:
                for t in of:
                    t.grad = None
                y.backward(dy)
                assert all(torch.equal(t.grad, b) for t, b in zip(of, want))
            else:
                assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, of, dy), want))


def test_saved_tensors_in_another_form_are_refused():
    x, w = leaf(matrix(37, 100, 1, torch.float16)), leaf(matrix(70, 100, 2, torch.float16))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:-1]):
        y = fp8.linear(x, w)
    with pytest.raises(RuntimeError, match="another form"):
        y.backward(torch.ones_like(y))


# ---- modules ----

def test_frozen_layers():
    lin = torch.nn.Linear(200, 131).half().cuda()
    q = fp8.Fp8Linear(lin)
    x = matrix(30, 200, 1, torch.float16)
    with torch.no_grad():
        y = q(x)
        check_product(y, value64(x), value64(lin.weight, square=True), lin.bias)
        assert torch.equal(q(x.reshape(2, 3, 5, 200)).reshape(30, 131), y)
        assert torch.equal(copy.deepcopy(q)(x), y)
        assert torch.equal(q.cpu().cuda()(x), y)
        other = fp8.Fp8Linear(torch.nn.Linear(200, 131).half().cuda())
        assert not torch.equal(other(x), y)
        other.load_state_dict(q.state_dict())
        assert torch.equal(other(x), y)
        other.load_state_dict({k: v.clone() for k, v in q.state_dict().items()}, assign=True)
        assert torch.equal(other(x), y)
        assert torch.equal(q.half()(x), y)
    assert torch.equal(q(x), y) and not q(x).requires_grad      # the bias is as frozen as the weight
    with pytest.raises(capi.VenomError, match="trainable"):
        q(leaf(x))


def test_frozen_mlp_and_conversion():
    net = torch.nn.Sequential(torch.nn.Linear(96, 200), torch.nn.GELU(), torch.nn.Linear(200, 72)).half().cuda().requires_grad_(False)
    x = matrix(45, 96, 1, torch.float16)
    m = fp8.Fp8Mlp(net[0], net[2])
    want = fp8.mlp(x, net[0].weight, net[0].bias, net[2].weight, net[2].bias)
    assert torch.equal(m(x), want) and torch.equal(m(x.reshape(5, 9, 96)).reshape(45, 72), want)
    conv = fp8.linear_to_fp8(copy.deepcopy(net))
    a = fp8.linear(x, net[0].weight, net[0].bias)
    assert torch.equal(conv[0](x), a) and torch.equal(conv(x), fp8.linear(torch.nn.functional.gelu(a), net[2].weight, net[2].bias))


def test_layers_in_files():
    import io
    x = matrix(30, 200, 1, torch.float16)
    fc, proj = torch.nn.Linear(200, 131).half().cuda(), torch.nn.Linear(131, 72).half().cuda()
    for layer in (fp8.Fp8Linear(fc), fp8.Fp8Mlp(fc, proj), fp8.Fp8Linear(fc, trainable=True)):
        with torch.no_grad():
            want = layer(x)                    # views of the bytes exist when it is written
            f = io.BytesIO()
            torch.save(layer, f)
            f.seek(0)
            assert torch.equal(torch.load(f, weights_only=False)(x), want) and torch.equal(copy.deepcopy(layer)(x), want)


def test_one_tensor_in_several_places():
    q = fp8.quantize(matrix(150, 260, 1, torch.float16))
    v = q.dequantize().double()
    y = fp8.matmul(q, q, dtype=torch.float32)
    assert bool(((y.double() - v @ v.t()).abs() <= 260 * 2.0 ** -23 * (v.abs() @ v.abs().t())).all())
    x, w, b = matrix(96, 96, 1, torch.float16), matrix(96, 96, 2, torch.float16), matrix(1, 96, 3, torch.float16)[0].clone()
    dy = matrix(96, 96, 9, torch.float16)
    # a weight and a bias that both layers share: the sum of what two of their own get
    apart = [leaf(t) for t in (x, w, b, w, b)]
    grads = torch.autograd.grad(fp8.mlp(*apart), apart, dy)
    x1, w1, b1 = leaf(x), leaf(w), leaf(b)
    got = torch.autograd.grad(fp8.mlp(x1, w1, b1, w1, b1), (x1, w1, b1), dy)
    assert torch.equal(got[0], grads[0]) and torch.equal(got[1], grads[1] + grads[3]) and torch.equal(got[2], grads[2] + grads[4])
    # one leaf as input and as weight
    apart = [leaf(x), leaf(x)]
    grads = torch.autograd.grad(fp8.linear(*apart), apart, dy)
    both = leaf(x)
    assert torch.equal(torch.autograd.grad(fp8.linear(both, both), both, dy)[0], grads[0] + grads[1])


def test_layers_in_inference_mode():
    lin, x = torch.nn.Linear(200, 131).half().cuda(), matrix(30, 200, 1, torch.float16)
    want = fp8.Fp8Linear(lin)(x)
    with torch.inference_mode():
        made = fp8.Fp8Linear(lin)
        assert torch.equal(made(x), want) and torch.equal(fp8.linear(x, lin.weight, lin.bias), want)
        assert torch.equal(fp8.quantize(x).dequantize(), value64(x).float())
    with torch.no_grad():
        assert torch.equal(made(x), want)


def test_gradients_accumulate_and_repeat():
    """Two calls of one layer in one graph, backward twice: gradients add up, and saved tensors are as they were."""
    x, w, b = leaf(matrix(50, 96, 1, torch.float16)), leaf(matrix(72, 96, 2, torch.float16)), leaf(matrix(1, 72, 3, torch.float16)[0].clone())
    dy = matrix(50, 72, 9, torch.float16)
    want = torch.autograd.grad(fp8.linear(x, w, b), (x, w, b), dy)
    y = fp8.linear(x, w, b)
    first = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    assert all(torch.equal(a, c) for a, c in zip(first, want))
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(y, (x, w, b), dy), want))
    (fp8.linear(x, w, b) + fp8.linear(x, w, b)).backward(dy)
    assert all(torch.equal(t.grad, c + c) for t, c in zip((x, w, b), want))


def test_training_step_with_modules():
    """Trainable modules share their parameters with the originals; a step changes the next call's result."""
    net = torch.nn.Sequential(torch.nn.Linear(96, 128), torch.nn.LayerNorm(128)).cuda()
    weight = net[0].weight
    fp8.linear_to_fp8(net, trainable=True)
    ff = fp8.Fp8Mlp(torch.nn.Linear(128, 256).cuda(), torch.nn.Linear(256, 128).cuda(), trainable=True)
    opt = torch.optim.SGD(list(net.parameters()) + list(ff.parameters()), lr=0.1)
    x = matrix(64, 96, 1)
    first = ff(net(x))
    first.square().mean().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in opt.param_groups[0]["params"])
    opt.step()
    assert net[0].weight is weight and not torch.equal(ff(net(x)), first)


def decoder(layers=2):
    from venom_b200 import e2e_gpt
    torch.manual_seed(3)
    with torch.device("cuda"):
        return e2e_gpt.build_block(layers, 256, 4, 1024).half()


def test_decoder_block_in_8_bits():
    """The command's block as a user runs it: forward frozen and trainable, a training step's gradients against the dense block's."""
    from venom_b200 import e2e_gpt
    dense = decoder()
    x, dy = matrix(2 * 96, 256, 1, torch.float16, 0.0).reshape(2, 96, 256), matrix(2 * 96, 256, 2, torch.float16, 0.0).reshape(2, 96, 256)
    with torch.no_grad():
        want = dense(x)
        frozen, trainable = e2e_gpt.to_fp8(dense), e2e_gpt.to_fp8(dense, trainable=True)
        got = frozen(x)
        assert torch.equal(got, trainable(x))
    # every linear's operands are off by 2^-4 at most and 2^-5.8 of a standard deviation on average (uniform over a step), two of them, in eight linears whose results
    # are added to the residual stream: 2^-5.8 sqrt(2 8) = 2^-3.8 of it if they were all as large as the stream
    assert (got.float() - want.float()).norm() <= 2.0 ** -3.8 * want.float().norm()
    # gradients: three operands more on their way, so below 2^-3 of their norm by the same count; a cosine of 0.9 would take 0.43
    g, w = e2e_gpt.train_step(trainable, x, dy), e2e_gpt.train_step(dense, x, dy)
    names = [n for n, _ in trainable.named_parameters()]
    assert len(g) == len(w) == len(names) + 1 and {id(p) for p in trainable.parameters()} == {id(p) for p in dense.parameters()}
    order = {id(p): i for i, p in enumerate(dense.parameters())}
    for p, got_p in zip(trainable.parameters(), g[1:]):
        ref = w[1 + order[id(p)]].float()
        assert got_p.isfinite().all() and torch.nn.functional.cosine_similarity(got_p.float().flatten(), ref.flatten(), dim=0) > 0.9
    assert torch.nn.functional.cosine_similarity(g[0].float().flatten(), w[0].float().flatten(), dim=0) > 0.9


def test_decoder_commands_run(capsys):
    from venom_b200 import e2e_gpt
    try:
        e2e_gpt.main(["--layers", "1", "--hidden", "256", "--heads", "4", "--ffn", "1024", "--batch", "2", "--seq", "64", "--repeats", "2", "-v", "64", "-m", "8", "--fp8", "--train"])
    finally:
        torch.set_grad_enabled(True)
    out = capsys.readouterr().out
    assert "fp8 forward," in out and "fp8 training step," in out and "dense training step," in out


# ---- streams, graphs, devices ----

def test_calls_on_another_stream():
    x, w = matrix(500, 1024, 1, torch.float16), matrix(768, 1024, 2, torch.float16)
    want = fp8.linear(x, w)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    with torch.cuda.stream(s):
        for _ in range(3):
            outs.append(fp8.linear(x, w))
    other = fp8.linear(x, w)          # both streams at once
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs + [other])


def test_captured_training_step():
    """Forward and backward captured into two graphs and replayed on new inputs.  While an eager graph of the same leaves lives the capture is refused: its nodes
    belong to the eager stream, and a capture that the backward pass takes there breaks."""
    leaves = block(130, 128, 256, 128, torch.float16)
    dy = matrix(130, 128, 9, torch.float16)
    eager = fp8.mlp(*leaves)
    y1, y2 = fp8.linear(leaves[0], leaves[1], leaves[2]), fp8.gelu(leaves[0])
    for call in (lambda: fp8.mlp(*leaves), lambda: fp8.linear(leaves[0], leaves[1]), lambda: fp8.gelu(leaves[0])):
        g = torch.cuda.CUDAGraph()
        with pytest.raises(capi.VenomError, match="still lives"):
            with torch.cuda.graph(g):
                call()
    with torch.no_grad():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plain = fp8.mlp(*leaves)
        g.replay()
        assert torch.equal(plain, eager)
    torch.autograd.grad(eager, leaves, dy)
    del eager, y1, y2
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(fp8.mlp(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    outs = []
    for g in (g1, g2):
        with torch.cuda.graph(g):
            y = fp8.mlp(*leaves)
            outs.append([y.detach()] + list(torch.autograd.grad(y, leaves, dy)))
            del y
    with torch.no_grad():
        leaves[0].copy_(matrix(130, 128, 77, torch.float16))
    want = fp8.mlp(*leaves)
    want = [want.detach()] + list(torch.autograd.grad(want, leaves, dy))
    g1.replay()
    g2.replay()
    g1.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_first_call_inside_a_capture():
    """A process whose first 8-bit calls are captured: what a device needs once is set up then."""
    code = """
import torch
from venom_b200 import fp8
x, w = torch.randn(300, 512, device="cuda").half(), torch.randn(700, 512, device="cuda").half()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = fp8.linear(x, w)
    t = fp8.quantize(x, both=True)[1]
g.replay()
assert torch.equal(y, fp8.linear(x, w)) and torch.equal(t.dequantize(), fp8.quantize(x, both=True)[1].dequantize())
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_calls_from_two_threads():
    import threading
    x, w = matrix(260, 1024, 1, torch.float16), matrix(520, 1024, 2, torch.float16)
    want = fp8.linear(x, w)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(50):
                if not torch.equal(fp8.linear(x, w), want):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
