"""Accuracy of the 8-bit operators' GELU and of its gradient, in every kernel that computes them: rows with a result of the input's type, rows and tiles of 128 x 128
with 8-bit results, their transposes, checkpoints and column sums.

The exact form is h = Phi(-a) = R(t) exp(-a^2 / 2), a = |x|, t = 1 / (1 + p a).  Its relative error, term by term, for results of 16-bit values (32-bit ones, derivatives): R's fit
1.45e-6 (3.3e-7); the exponential 2^-22, its argument twice rounded, a^2 / 2 2^-23; the reciprocal 2^-23 and its argument 2^-24, times at most 2.7 (3.2), the elasticity of R(t);
coefficients and steps of R, whose terms are at most 1.7 (2.2) times the sum, 2 * 1.7 * 2^-24; a product 2^-24: 2.5e-6 (1.6e-6) + a^2 2^-24 in all.  The tanh form is x / (1 + exp(-2 u)): the exponential 2^-22, its argument |2 u log2 e| three times
rounded and its constants once, so |u| 2^-21, sum, reciprocal and product 2^-22: 1e-6 + |u| 2^-21.  u = sqrt(2 / pi) (a + 0.044715 a^3).  A tail or an exponential
below 2^-126 may be flushed to zero, which takes 2^-126 times what it is multiplied with from a result."""
import math

import pytest
import torch

from test_fp8_gpu import E4M3, E5M2, TYPES, exponent, gelu64, matrix, pow2, unpacked, value64
from venom_b200 import capi, fp8

pytestmark = pytest.mark.gpu
CODES = {"fp32": 0, "fp16": 1, "bf16": 2}
NORMAL = 2.0 ** -126


def form_error(a, tanh, fine):
    """Relative error of what decays with |x|: Phi(-|x|) or 1 / (1 + exp(2 |u|))."""
    return 1e-6 + math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3) * 2.0 ** -21 if tanh else (1.6e-6 if fine else 2.5e-6) + a * a * 2.0 ** -24


def gelu_parts(x, tanh, dtype):
    """(GELU, its derivative, bounds of their errors in 32 bits) in 64 bits, without cancellation for x < 0."""
    x = x.double()
    a = x.abs().clamp(max=64.0)
    rel, rel_d = form_error(a, tanh, dtype == "fp32"), form_error(a, tanh, True)
    if tanh:
        u = math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
        h = torch.sigmoid(-2 * u)
        du = 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * a ** 2)
        slope = a * h * torch.sigmoid(2 * u) * du
    else:
        h, du = 0.5 * torch.special.erfc(a * math.sqrt(0.5)), 1.0
        slope = a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    y = x.clamp(min=0) - a * h
    d = torch.where(x < 0, h - slope, 1 - h + slope)
    # the positive side is x - a h or x (1 - h), one rounding more of each; the derivative a sum of h, 1 and the slope: x h (1 - h) du with h twice and four roundings more, or
    # the exponential with one rounded constant more in its argument
    ey = rel * a * h + torch.where(x < 0, 0.0, 2.0 ** -22 * x.abs())
    ed = rel_d * h + (rel_d * (2.0 if tanh else 1.0) + 2.0 ** -22 + a * a * 2.0 ** -24) * slope + 2.0 ** -23 * torch.where(x < 0, h + slope, 1.0 + slope)
    return y, d, ey + (1 + a) * NORMAL, ed + (1 + a * du) * NORMAL


def within(got, want, error):
    """Rounded once to the type of `got` from a value that is off by at most `error`."""
    info = torch.finfo(got.dtype)
    bound = error + info.eps / 2 * (want.abs() + error) + info.smallest_normal * info.eps / 2
    far = ((got.double() - want).abs() - bound).nan_to_num(nan=1.0)
    assert not bool((far > 0).any()), "%g over the bound, at %s" % (far.max().item(), far.flatten().argmax().item())


def grid(dtype):
    """Every region of the function: 0, both tails as far as they reach, the zero of the derivative."""
    x = torch.cat([torch.linspace(-14, 14, 28001, dtype=torch.float64), torch.linspace(-1, 1, 4001, dtype=torch.float64), torch.logspace(-30, 1, 300, dtype=torch.float64),
                   -torch.logspace(-30, 1, 300, dtype=torch.float64)])
    return torch.cat([x, x.new_zeros(-len(x) % 512)]).to(TYPES[dtype]).cuda().view(-1, 512)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tanh", [False, True])
def test_values(dtype, tanh):
    x = grid(dtype)
    y, _, error, _ = gelu_parts(x, tanh, dtype)
    within(fp8.gelu(x, "tanh" if tanh else "none"), y, error)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tanh", [False, True])
def test_derivatives(dtype, tanh):
    """At the values that a checkpoint can hold: all of e4m3 in blocks of their own, with scales from 2^-11 to 1."""
    units = torch.arange(256, dtype=torch.uint8, device="cuda").view(E4M3).float()
    units = units[units.isfinite()]
    h = torch.cat([units * 2.0 ** -e for e in range(12)])
    h = h[h.abs() < 14][:, None].expand(-1, 128).contiguous()
    dy = matrix(*h.shape, 3, TYPES[dtype])
    x = h.to(TYPES[dtype]).requires_grad_()                # exact: four bits, 2^-21 at least
    assert torch.equal(x.detach().float(), h)
    (dx,) = torch.autograd.grad(fp8.gelu(x, "tanh" if tanh else "none"), x, dy)
    assert torch.equal(fp8.quantize(h).dequantize(), h)
    _, d, _, error = gelu_parts(h, tanh, dtype)
    within(dx, dy.double() * d, dy.double().abs() * error)
    at_zero = h == 0
    assert bool(at_zero.any()) and torch.equal(dx[at_zero], dy[at_zero] * 0.5)          # to the last bit
    # and against differences: half a third derivative (below 2) times d^2, and 64 bits' own rounding of the two values
    step = 1e-5
    slope = (gelu64(h.double() + step, tanh)[0] - gelu64(h.double() - step, tanh)[0]) / (2 * step)
    assert bool(((slope - d).abs() <= step ** 2 + 2.0 ** -52 * (1 + h.double().abs()) / step).all())


def held_within(q, want, error, f8, doubtful=None):
    """8 bits of values that are off by at most `error`: the scale is that of the largest magnitude, or next to it where the error reaches over the line, and the
    value one of those that a value within the error may be rounded to.  `want` may hold NaN and infinities, which of them where `doubtful` is left open."""
    top, low, bits = (448.0, -6, 3) if f8 == E4M3 else (57344.0, -14, 2)
    got, e = unpacked(q)
    n, k = want.shape
    finite = want.isfinite()
    size, slack = (torch.where(finite, t, torch.zeros_like(t)) for t in (want.abs(), error))
    pad = (0, -k % 128)
    blocks = lambda t: torch.nn.functional.pad(t, pad).view(n, -1, 128).amax(-1)

    def code(amax):
        c = torch.where(amax > 0, exponent(amax.clamp(min=1e-300)) - exponent(torch.tensor(top, dtype=torch.float64)).item(), torch.full_like(amax, -127)).clamp(min=-127)
        return torch.where(amax > top * pow2(c), c + 1, c)

    assert bool(((e >= code(blocks((size - slack).clamp(min=0)))) & (e <= code(blocks(size + slack)))).all()), "scales"
    s = pow2(e).repeat_interleave(128, 1)[:, :k]
    step = pow2(exponent(((size + slack) / s).clamp(min=2.0 ** low)) - bits) * s
    off = (got * s - want).abs()
    assert bool(((off <= step / 2 + slack) | ~finite).all()), "values"
    kept = want if f8 == E5M2 else torch.where(want.isinf(), math.nan, want)
    assert not bool(got[~finite].isfinite().any())
    sure = ~finite if doubtful is None else ~finite & ~doubtful
    assert torch.equal(got[sure].nan_to_num(nan=1e9), kept[sure].nan_to_num(nan=1e9)), "values that are not finite"


def packed(rows, cols, f8=E4M3):
    """Room for a matrix in 8 bits that holds neither zeros nor numbers."""
    ld = -(-cols // 16) * 16
    data = torch.full((rows, ld), 0xFF, dtype=torch.uint8, device="cuda")
    return fp8.BlockFp8(data.view(f8)[:, :cols], torch.full((-(-cols // 512), rows, 4), 0xFF, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))


def room(q):
    return [None, 16, None] if q is None else [q.data.data_ptr(), q.data.stride(0), q.scales.data_ptr()]


def troubled(rows, cols, dtype, seed, lowest):
    """Normal values with the ones that go wrong: NaN, infinities, the lowest value as a mask writes it, rows of zeros, whole blocks that are not finite."""
    x = matrix(rows, cols, seed, TYPES[dtype], 0.7)
    x[0] = 0
    if rows > 40:
        x[1] = lowest
        x[5, 3 % cols], x[9, -1], x[11, cols // 2] = math.nan, math.inf, -math.inf
        x[12:20] = -math.inf                            # whole patches of a thread
        x[24:28] = math.nan
        x[32] = math.inf
    return x


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 40), (129, 257), (256, 256), (300, 777)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tanh", [False, True])
def test_8_bit_results(rows, cols, dtype, tanh):
    """vnm_fp8_gelu: rows alone, both orientations, each alone, with and without a checkpoint; all of them alike."""
    x = troubled(rows, cols, dtype, 5, torch.finfo(TYPES[dtype]).min)
    want, _, error, _ = gelu_parts(x, tanh, dtype)
    want = torch.where(x == -math.inf, torch.zeros_like(want), torch.where(x == math.inf, math.inf, want))
    want = torch.where(x.isnan(), math.nan, want)
    stream, results = torch.cuda.current_stream().cuda_stream, []
    for by_rows, transposed, checkpoint in ((1, 0, 0), (1, 0, 1), (1, 1, 0), (1, 1, 1), (0, 1, 1)):
        q, t, c = (packed(rows, cols) if by_rows else None, packed(cols, rows) if transposed else None, packed(rows, cols) if checkpoint else None)
        assert capi.lib().vnm_fp8_gelu(x.data_ptr(), CODES[dtype], cols, rows, cols, tanh, None, cols, *room(q), *room(t), *room(c), stream) == 0
        results.append((q, t, c))
        if q is not None:
            held_within(q, want, error, E4M3)
        if t is not None:
            held_within(t, want.t(), error.t(), E4M3)
        if c is not None:
            ref = fp8.quantize(x)
            assert torch.equal(c.data.view(torch.uint8), ref.data.view(torch.uint8)) and torch.equal(c.scales.view(torch.uint8), ref.scales.view(torch.uint8))
    for i in (0, 1):
        kept = [r[i] for r in results if r[i] is not None]
        assert all(torch.equal(k.data.view(torch.uint8), kept[0].data.view(torch.uint8)) and torch.equal(k.scales.view(torch.uint8), kept[0].scales.view(torch.uint8)) for k in kept)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 40), (129, 257), (256, 256), (300, 777)])
@pytest.mark.parametrize("dtype,f8", [("fp16", E4M3), ("bf16", E5M2), ("fp32", E4M3), ("fp32", E5M2)])
@pytest.mark.parametrize("tanh", [False, True])
def test_8_bit_gradients(rows, cols, dtype, f8, tanh):
    """vnm_fp8_gelu_grad: rows alone, both orientations, each alone; column sums."""
    dy = troubled(rows, cols, dtype, 6, -60000.0)
    h = matrix(rows, cols, 7, spread=0.7) + 1.0
    ckpt = fp8.quantize(h)
    _, d, _, error = gelu_parts(value64(h), tanh, dtype)
    doubtful = d.abs() <= error            # may come out as 0, and 0 times an infinity is NaN
    want, error = dy.double() * d, dy.double().abs() * error + 2.0 ** -24 * (dy.double() * d).abs() + NORMAL
    stream, lib = torch.cuda.current_stream().cuda_stream, capi.lib()
    code, results = (0 if f8 == E4M3 else 1), []
    for by_rows, transposed, sums in ((1, 0, 0), (1, 1, 0), (1, 1, 1), (0, 1, 1)):
        q, t = packed(rows, cols, f8) if by_rows else None, packed(cols, rows, f8) if transposed else None
        total = torch.full((cols,), 7.0, device="cuda") if sums else None
        ws = torch.empty(-(-rows // 128) * cols, device="cuda") if sums else None
        assert lib.vnm_fp8_gelu_grad(dy.data_ptr(), CODES[dtype], cols, rows, cols, tanh, *room(ckpt), None, cols, code, *room(q), *room(t), total.data_ptr() if sums else None, 0,
                                     ws.data_ptr() if sums else None, stream) == 0
        results.append((q, t))
        if q is not None:
            held_within(q, want, error, f8, doubtful)
        if t is not None:
            held_within(t, want.t(), error.t(), f8, doubtful.t())
        if sums:
            exact = want.sum(0)
            fine = exact.isfinite()
            bound = error.sum(0) + rows * 2.0 ** -23 * want.abs().sum(0)
            assert bool(((total.double() - exact).abs() <= bound)[fine].all()) and torch.equal(total.isnan() & exact.isnan(), exact.isnan())
    for i in (0, 1):
        kept = [r[i] for r in results if r[i] is not None]
        assert all(torch.equal(k.data.view(torch.uint8), kept[0].data.view(torch.uint8)) and torch.equal(k.scales.view(torch.uint8), kept[0].scales.view(torch.uint8)) for k in kept)
