"""Linears in block-scaled 8 bits, with 8-bit activation checkpoints for their backward pass.

What nmv.SrnmSpmm is for a weight that may be pruned, Fp8Linear is for one that may not: every value is kept, in 8 bits, with a power of
two for each block of 128 along a row (for each 128 x 128 of a weight).  The product's operands are both in that form and are scaled inside the tensor
core; sums have 32 bits.  For training, what a layer keeps of its input until the backward pass is 8 bits a value too: the transpose that the weight's
gradient multiplies with, written in the same pass as the operand of the forward product.

  quantize, BlockFp8         the format and its conversions (capi.compress and decompress of this form)
  matmul                     a @ b.T of two of them
  linear, gelu, mlp          differentiable: linear layer, GELU from an 8-bit checkpoint, and linear - GELU - linear with the GELU between them fused into
                             the quantiser, forwards and backwards
  Fp8Linear, Fp8Mlp, linear_to_fp8   modules, as nmv.SrnmSpmm and nmv.linear_to_spmm

Everything runs on the CUDA device of its operands and on torch's current stream there; nothing synchronises, and calls may be captured into a graph.
There is no CPU path.
"""
import torch

from . import spatha_module
from .capi import VenomError

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)

_ext = None


def _load():
    global _ext
    _ext = spatha_module()
    return _ext


def _error(e):
    return VenomError(str(e).split("\nException raised from")[0])


def _call(name, *args):
    try:
        return getattr(_ext or _load(), name)(*args)
    except (RuntimeError, TypeError) as e:
        raise _error(e) from None


class BlockFp8:
    """A matrix in 8 bits: `data` float8_e4m3fn or float8_e5m2 [rows, cols], rows a multiple of 16 bytes apart, and `scales` float8_e8m0fnu
    [ceil(cols / 512), rows, 4]: scales[kb // 4, r, kb % 4] is that of columns 128 kb .. 128 kb + 127 of row r.  Both are used as they lie."""

    __slots__ = ("data", "scales")

    def __init__(self, data, scales):
        self.data, self.scales = data, scales

    @property
    def shape(self):
        return self.data.shape

    @property
    def dtype(self):
        return self.data.dtype

    @property
    def device(self):
        return self.data.device

    def dequantize(self, dtype=torch.float32):
        """The values that it stands for, [rows, cols] of `dtype` (float16, bfloat16 or float32)."""
        return _call("fp8_dequantize", self.data, self.scales, dtype)

    def __repr__(self):
        return "BlockFp8(%d x %d, %s, %s)" % (self.shape[0], self.shape[1], self.dtype, self.device)


def quantize(x, dtype=E4M3, square=False, both=False):
    """x [rows, cols] (float16, bfloat16 or float32 on a CUDA device) -> BlockFp8 of float8_e4m3fn or float8_e5m2.

    A block's scale is the smallest power of two that brings its largest finite magnitude to at most 448 (e4m3) or 57344 (e5m2); values are
    rounded to nearest even.  NaN stays NaN, infinities become NaN in e4m3 and stay in e5m2.  Not differentiable: the result is x's values now.  Blocks are 128 values of a row, or with `square` 128 x 128,
    so that a matrix and its transpose hold the same values.  both: also the transpose, as (BlockFp8 of x, BlockFp8 of x.T), from one read of x."""
    try:
        q = (_ext or _load()).fp8_quantize(x, dtype, bool(square), bool(both))
    except (RuntimeError, TypeError) as e:
        raise _error(e) from None
    return (BlockFp8(q[0], q[1]), BlockFp8(q[2], q[3])) if both else BlockFp8(*q)


def matmul(a, b, bias=None, dtype=torch.float16):
    """a @ b.T (+ bias): BlockFp8 [M, K] and [N, K] -> [M, N] of `dtype` (float16, bfloat16 or float32).  The 8-bit types of a and b may differ.
    bias: N values, added in 32 bits.  Not differentiable: the result belongs to no graph, also where the bias wants a gradient (linear is).  Sums have 32 bits, as
    the tensor core keeps them: they are truncated, not rounded, and zero below 2^-126."""
    try:
        return (_ext or _load()).fp8_matmul(a.data, a.scales, b.data, b.scales, bias, dtype)
    except (RuntimeError, TypeError) as e:
        raise _error(e) from None


def _check_input(x, what):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise VenomError("%s: a CUDA tensor expected (there is no CPU path)" % what)
    if x.dtype not in _FLOATS:
        raise VenomError("%s: float16, bfloat16 or float32 expected, not %s" % (what, x.dtype))
    if x.dim() < 1:
        raise VenomError("%s: at least one dimension expected" % what)


def _check_grad_dtype(grad_dtype, what):
    if grad_dtype not in (E4M3, E5M2):
        raise VenomError("%s: gradients are kept in float8_e4m3fn or float8_e5m2, not %s" % (what, grad_dtype))


def _tanh_form(approximate, what):
    if approximate not in ("none", "tanh"):
        raise VenomError("%s: approximate is 'none' or 'tanh', not %r" % (what, approximate))
    return approximate == "tanh"


def linear(x, weight, bias=None, grad_dtype=E4M3):
    """x @ weight.T + bias for x [..., in], weight [out, in] and bias [out], differentiable once in all three; the result has the type of x, gradients
    have their inputs' types.

    x is rounded in blocks of 128 along its features, the weight in blocks of 128 x 128, gradients in blocks of 128 of `grad_dtype` (float8_e4m3fn
    or float8_e5m2) along whichever way they are summed; the bias's gradient is the sum of unrounded ones.  Kept until the backward pass: the 8-bit
    transpose of x (where the weight wants a gradient), and of the weight (where x does) what takes less: its 8-bit transpose where it has no more rows than x has
    tokens, another type than x, or is not a leaf; else the weight itself, which may not be written to meanwhile."""
    return _call("fp8_linear", x, weight, bias, grad_dtype)


def gelu(x, approximate="none"):
    """GELU of x [..., features] like torch.nn.functional.gelu, but 0 for -inf; what is kept for the backward pass is x in 8 bits, in blocks of 128
    features.  For negative x the result is off by 2.5e-6 (32-bit x: 1.6e-6) + x^2 2^-24 of itself at most, besides its rounding (the tanh form, with u its argument: 1e-6 + |u| 2^-21)."""
    return _call("fp8_gelu8", x, _tanh_form(approximate, "fp8.gelu"))


def mlp(x, w1, b1, w2, b2, approximate="none", grad_dtype=E4M3):
    """linear(gelu(linear(x, w1, b1)), w2, b2) for x [..., in], w1 [hidden, in], w2 [out, hidden], differentiable once in all five.

    The GELU's result is rounded to 8 bits straight from 32 (there is no copy of it in the type of x), its gradient likewise.  Kept until the
    backward pass, in 8 bits: the transposes of x and of the GELU's result, and the GELU's input; the weights as in linear."""
    return _call("fp8_mlp", x, w1, b1, w2, b2, _tanh_form(approximate, "fp8.mlp"), grad_dtype)


def _autocast(x):
    """What torch.nn.Linear would multiply: under torch.autocast x in the type that is named there."""
    if torch.is_autocast_enabled("cuda") and isinstance(x, torch.Tensor) and x.dtype in _FLOATS:
        return x.to(torch.get_autocast_dtype("cuda"))
    return x


class _Held(torch.nn.Module):
    """A frozen weight's 8 bits as buffers.  They are kept as bytes, which Module.half() and its like leave alone, with the rows' padding, which a copy to
    another device would drop; the padding is zero, so that one weight always gives the same bytes."""

    def _hold(self, name, weight):
        q = quantize(weight.detach(), square=True)
        rows, cols = q.shape
        data = torch.zeros((rows, max(16, -(-cols // 16) * 16)), dtype=torch.uint8, device=q.device)
        data[:, :cols] = q.data.view(torch.uint8)
        self.register_buffer(name + "_data", data)
        self.register_buffer(name + "_scales", q.scales.view(torch.uint8).clone())      # storages of their own, as files want them
        self._cols[name] = cols

    def __setstate__(self, state):
        state = dict(state)
        if "_views" in state:      # of files that kept views beside the buffers
            state["_cols"] = {name: view[0] for name, view in state.pop("_views").items()}
        super().__setstate__(state)

    def _weight(self, name):
        """The bytes that the buffers hold now, their scales, and the columns that they stand for."""
        return self._buffers[name + "_data"], self._buffers[name + "_scales"], self._cols[name]

    def _refuse_gradients(self, x):
        if torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad:
            raise VenomError("%s holds a frozen weight: build it with trainable=True for gradients" % type(self).__name__)


def _frozen(bias):
    """The same values as a parameter that wants no gradient."""
    return None if bias is None else torch.nn.Parameter(bias.detach(), requires_grad=False)


class Fp8Linear(_Held):
    """Drop-in replacement of torch.nn.Linear whose products run in 8 bits; results have the type of the input, under torch.autocast the type that it names.

    trainable=False: the weight is quantised once and held in 8 bits only, like SrnmSpmm's, for inference; an input that wants a gradient is refused.  trainable=True: the layer keeps the parameters
    of `original`, quantises the weight in every call and is differentiable (see linear)."""

    def __init__(self, original, trainable=False, grad_dtype=E4M3):
        super().__init__()
        self._cols = {}
        _check_grad_dtype(grad_dtype, "Fp8Linear")
        self.in_features, self.out_features = original.in_features, original.out_features
        self.trainable, self.grad_dtype = bool(trainable), grad_dtype
        self.bias = original.bias if self.trainable else _frozen(original.bias)
        if self.trainable:
            self.weight = original.weight
        else:
            _check_input(original.weight, "Fp8Linear")
            self._hold("weight", original.weight)

    def forward(self, input):
        if self.trainable:
            return linear(_autocast(input), self.weight, self.bias, self.grad_dtype)
        self._refuse_gradients(input)
        return _call("fp8_held_linear", _autocast(input), *self._weight("weight"), self.bias)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, bias=%s, trainable=%s" % (self.in_features, self.out_features, self.bias is not None, self.trainable)


class Fp8Mlp(_Held):
    """The feed-forward block proj(gelu(fc(x))) of two torch.nn.Linear in 8 bits, the GELU fused into the quantiser (see mlp).  trainable as in Fp8Linear."""

    def __init__(self, fc, proj, approximate="none", trainable=False, grad_dtype=E4M3):
        super().__init__()
        self._cols = {}
        _check_grad_dtype(grad_dtype, "Fp8Mlp")
        if fc.out_features != proj.in_features:
            raise VenomError("Fp8Mlp: %d features do not match %d" % (fc.out_features, proj.in_features))
        self.tanh_form, self.approximate = _tanh_form(approximate, "Fp8Mlp"), approximate
        self.trainable, self.grad_dtype = bool(trainable), grad_dtype
        self.out_features = proj.out_features
        self.fc_bias, self.proj_bias = (fc.bias, proj.bias) if self.trainable else (_frozen(fc.bias), _frozen(proj.bias))
        if self.trainable:
            self.fc_weight, self.proj_weight = fc.weight, proj.weight
        else:
            _check_input(fc.weight, "Fp8Mlp")
            _check_input(proj.weight, "Fp8Mlp")
            self._hold("fc", fc.weight)
            self._hold("proj", proj.weight)

    def forward(self, input):
        if self.trainable:
            return mlp(_autocast(input), self.fc_weight, self.fc_bias, self.proj_weight, self.proj_bias, self.approximate, self.grad_dtype)
        self._refuse_gradients(input)
        return _call("fp8_held_mlp", _autocast(input), *self._weight("fc"), self.fc_bias, *self._weight("proj"), self.proj_bias, self.tanh_form)


def linear_to_fp8(mod, skip=(), trainable=False, grad_dtype=E4M3):
    """Replaces every torch.nn.Linear below `mod` by Fp8Linear, but for the names in `skip` (nmv.linear_to_spmm's walk).

    Subclasses stay as they are: they compute something else, or their owner multiplies with their weight itself (torch.nn.MultiheadAttention.out_proj).  A
    torch.nn.TransformerEncoderLayer is kept from the fused inference path that takes its linears' weights past them."""
    if type(mod) is torch.nn.Linear:
        return Fp8Linear(mod, trainable, grad_dtype)
    for name, child in mod.named_children():
        if name in skip:
            continue
        if type(child) is torch.nn.Linear:
            setattr(mod, name, Fp8Linear(child, trainable, grad_dtype))
        else:
            linear_to_fp8(child, skip, trainable, grad_dtype)
    if isinstance(mod, torch.nn.TransformerEncoderLayer) and any(isinstance(child, Fp8Linear) for child in mod.children()):
        mod.activation_relu_or_gelu = 0
    return mod


def device_status():
    """0, or VenomError if a bounded device-side wait of an 8-bit product on the current device has given up since the last call (its result is then
    void).  Synchronises the current stream."""
    return _call("fp8_device_status")
