"""The block-scaled 8-bit operators without a GPU: what they refuse, and the sizes of the format."""
import ctypes as C

import pytest
import torch

from venom_b200 import capi, fp8

F32, F16, BF16, E4M3, E5M2 = 0, 1, 2, 0, 1
BAD, UNSUPPORTED = 1, 3


@pytest.fixture(scope="module")
def lib():
    from venom_b200 import build
    build.build_lib()
    return capi.lib()


@pytest.mark.parametrize("rows,cols,want", [(1, 1, 4), (1, 512, 4), (1, 513, 8), (3, 128, 12), (4096, 1024, 32768), (0, 5, 0), (5, 0, 0), (2 ** 31 - 1, 2 ** 31 - 1, (2 ** 31 - 1) * 4 * 2 ** 22)])
def test_bytes_of_scales(lib, rows, cols, want):
    assert lib.vnm_fp8_scale_bytes(rows, cols) == want


# Addresses that are never read: every call below is refused before it reaches the device.
X, Y, S = 0x10000, 0x20000, 0x30000


def quantize(lib, x=X, x_type=F16, ldx=64, rows=8, cols=64, f8=E4M3, data=Y, ldd=64, scales=S, data_t=None, ldt=16, scales_t=None, colsum=None, sum_type=F32, ws=None):
    return lib.vnm_fp8_quantize(x, x_type, ldx, rows, cols, f8, 0, data, ldd, scales, data_t, ldt, scales_t, colsum, sum_type, ws, None)


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), b"negative"), (dict(x_type=7), b"unknown type"), (dict(x=None), b"null"), (dict(ldx=63), b"leading dimension"), (dict(x=X + 1), b"aligned to its type"),
    (dict(f8=2), b"8-bit type"), (dict(scales=None), b"both values and scales"), (dict(ldd=56), b"16 bytes"), (dict(ldd=72), b"16 bytes"), (dict(data=Y + 8), b"16-byte boundary"),
    (dict(scales=S + 2), b"4-byte"), (dict(data=None, scales=None), b"nothing is wanted"), (dict(data_t=Y, scales_t=S, ldt=0), b"transpose"),
    (dict(colsum=Y, ws=X), b"workspace and the transpose"), (dict(colsum=Y, data_t=Y, scales_t=S), b"workspace"), (dict(colsum=Y, sum_type=9), b"column sums"),
])
def test_quantize_refuses(lib, change, message):
    assert quantize(lib, **change) == BAD
    assert message in lib.vnm_last_error_string()


def test_quantize_refuses_what_no_launch_can_index(lib):
    big = 2 ** 31 - 1
    assert quantize(lib, rows=big, cols=big, ldx=big, ldd=2 ** 31) == UNSUPPORTED


def test_products_that_no_launch_can_index(lib):
    big = 2 ** 31 - 1
    assert matmul(lib, M=big, N=big, ldo=big) == UNSUPPORTED
    assert lib.vnm_fp8_matmul_config(big, big, 64, F16, 1, 0, None, None, None, None) == UNSUPPORTED
    assert lib.vnm_fp8_matmul_config(8, 8, big, F16, 1, 0, None, None, None, None) == UNSUPPORTED


def test_empty_matrices_are_no_work(lib):
    assert quantize(lib, rows=0) == 0
    assert quantize(lib, cols=0) == 0
    assert lib.vnm_fp8_dequantize(None, 16, None, E4M3, 0, 8, None, F16, 8, None) == 0
    assert lib.vnm_fp8_gelu(None, F16, 8, 0, 8, 0, None, 8, None, 16, None, None, 16, None, None, 16, None, None) == 0
    assert lib.vnm_fp8_matmul(None, 16, None, E4M3, None, 16, None, E4M3, 0, 8, 8, None, F16, None, F16, 8, None) == 0


def matmul(lib, a=X, lda=64, sa=S, at=E4M3, b=Y, ldb=64, sb=S, bt=E5M2, M=4, N=8, K=64, bias=None, bias_type=F16, out=X, out_type=F16, ldo=8):
    return lib.vnm_fp8_matmul(a, lda, sa, at, b, ldb, sb, bt, M, N, K, bias, bias_type, out, out_type, ldo, None)


@pytest.mark.parametrize("change,message", [
    (dict(K=0), b"K at least 1"), (dict(M=-1), b"negative"), (dict(at=5), b"8-bit type"), (dict(out_type=4), b"type of the result"), (dict(bias=X, bias_type=3), b"bias"),
    (dict(a=None), b"null"), (dict(sb=None), b"both values and scales"), (dict(lda=48), b"16 bytes"), (dict(ldb=65), b"16 bytes"), (dict(a=X + 8), b"16-byte boundary"),
    (dict(ldo=7), b"leading dimension"), (dict(out=X + 1), b"alignment"), (dict(bias=X + 1), b"bias is not aligned"),
])
def test_matmul_refuses(lib, change, message):
    assert matmul(lib, **change) == BAD
    assert message in lib.vnm_last_error_string()


def test_matmul_refuses_what_no_launch_can_index(lib):
    big = 2 ** 31 - 300
    assert matmul(lib, M=big, N=big, ldo=big) == UNSUPPORTED


def gelu(lib, y=X, ldy=64, data=None, scales=None, data_t=None, scales_t=None, ckpt=None, ckpt_scales=None, ldc=64):
    return lib.vnm_fp8_gelu(X, F16, 64, 8, 64, 0, y, ldy, data, 64, scales, data_t, 16, scales_t, ckpt, ldc, ckpt_scales, None)


@pytest.mark.parametrize("change,code,message", [
    (dict(y=None), BAD, b"nothing is wanted"), (dict(ldy=60), BAD, b"leading dimension"), (dict(data=Y), BAD, b"both"), (dict(data_t=Y, scales_t=S), UNSUPPORTED, b"together with a transpose"),
    (dict(ckpt=Y), BAD, b"checkpoint"), (dict(ckpt=Y, ckpt_scales=S, ldc=60), BAD, b"checkpoint"),
])
def test_gelu_refuses(lib, change, code, message):
    assert gelu(lib, **change) == code
    assert message in lib.vnm_last_error_string()


def gelu_grad(lib, ckpt=Y, ckpt_scales=S, dx=X, f8=E4M3, data=None, scales=None, data_t=None, scales_t=None, colsum=None, ws=None):
    return lib.vnm_fp8_gelu_grad(X, F16, 64, 8, 64, 0, ckpt, 64, ckpt_scales, dx, 64, f8, data, 64, scales, data_t, 16, scales_t, colsum, F32, ws, None)


@pytest.mark.parametrize("change,code,message", [
    (dict(ckpt=None, ckpt_scales=None), BAD, b"no checkpoint"), (dict(ckpt_scales=None), BAD, b"checkpoint"), (dict(dx=None), BAD, b"nothing is wanted"), (dict(f8=3), BAD, b"8-bit type"),
    (dict(data_t=Y, scales_t=S), UNSUPPORTED, b"together with a transpose"), (dict(colsum=X, ws=Y), BAD, b"workspace and the transpose"),
])
def test_gelu_grad_refuses(lib, change, code, message):
    assert gelu_grad(lib, **change) == code
    assert message in lib.vnm_last_error_string()


def test_cpu_tensors_are_rejected():
    x, w = torch.zeros(4, 8), torch.zeros(16, 8)
    q = fp8.BlockFp8(torch.zeros(4, 16).to(torch.float8_e4m3fn), torch.zeros((1, 4, 4), dtype=torch.uint8).view(torch.float8_e8m0fnu))
    for call in (lambda: fp8.quantize(x), lambda: fp8.matmul(q, q), lambda: q.dequantize(), lambda: fp8.linear(x, w), lambda: fp8.gelu(x),
                 lambda: fp8.mlp(x, w, None, torch.zeros(8, 16), None), lambda: fp8.Fp8Linear(torch.nn.Linear(8, 16)),
                 lambda: fp8.Fp8Linear(torch.nn.Linear(8, 16), trainable=True)(x)):
        with pytest.raises(capi.VenomError, match="CUDA"):
            call()


def test_modules_refuse_what_does_not_fit():
    with pytest.raises(capi.VenomError, match="do not match"):
        fp8.Fp8Mlp(torch.nn.Linear(8, 16), torch.nn.Linear(8, 16), trainable=True)
    with pytest.raises(capi.VenomError, match="approximate"):
        fp8.Fp8Mlp(torch.nn.Linear(8, 16), torch.nn.Linear(16, 8), approximate="fast", trainable=True)
    with pytest.raises(capi.VenomError, match="gradients are kept"):
        fp8.Fp8Linear(torch.nn.Linear(8, 16), trainable=True, grad_dtype=torch.float16)


def test_linear_to_fp8_walks_like_linear_to_spmm():
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.head = torch.nn.Linear(8, 16), torch.nn.Linear(16, 4)
            self.inner = torch.nn.Sequential(torch.nn.Linear(16, 16), torch.nn.ReLU())

    b = Block()
    weight = b.a.weight
    assert fp8.linear_to_fp8(b, skip=("head",), trainable=True) is b
    assert isinstance(b.a, fp8.Fp8Linear) and b.a.weight is weight and isinstance(b.inner[0], fp8.Fp8Linear) and type(b.head) is torch.nn.Linear
    assert {n for n, _ in b.named_parameters()} == {"a.weight", "a.bias", "head.weight", "head.bias", "inner.0.weight", "inner.0.bias"}
    assert isinstance(fp8.linear_to_fp8(torch.nn.Linear(8, 8), trainable=True), fp8.Fp8Linear)


def test_linear_to_fp8_leaves_subclasses():
    class Doubled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    attention = torch.nn.MultiheadAttention(8, 2)
    projection = attention.out_proj
    b = torch.nn.ModuleDict({"attention": attention, "own": Doubled(8, 8), "plain": torch.nn.Linear(8, 8)})
    own = b["own"]
    fp8.linear_to_fp8(b, trainable=True)
    assert attention.out_proj is projection and b["own"] is own and isinstance(b["plain"], fp8.Fp8Linear)
    assert fp8.linear_to_fp8(own, trainable=True) is own
