"""The block-scaled 8-bit operators where values are not finite, buffers change hands and memory counts."""
import copy
import math

import pytest
import torch

from test_fp8_gpu import E4M3, E5M2, TYPES, check_held, matrix, pow2
from venom_b200 import capi, fp8

pytestmark = pytest.mark.gpu


# ---- values that are not finite ----

def rows_of_nan(x):
    x[140:144] = math.nan                      # four rows that one thread of each sixteen holds


def patch_of_nan(x):
    x[8:12, 16:24] = math.nan                  # all that one thread holds


def patch_beside_an_infinity(x):
    x[8:12, 16:24], x[13, 100] = math.nan, -math.inf


def tile_of_nan(x):
    x[128:256, :128] = math.nan


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("f8", [E4M3, E5M2])
@pytest.mark.parametrize("where", [rows_of_nan, patch_of_nan, patch_beside_an_infinity, tile_of_nan])
@pytest.mark.parametrize("square", [False, True])
def test_nan_side_by_side_leaves_the_other_values(dtype, f8, where, square):
    """The largest finite value of a tile lies in the eight rows that a warp holds together with the NaN."""
    x = matrix(260, 300, 3, TYPES[dtype], 0.5)
    x[14, 30], x[137, 250], x[139, 20] = 1000.0, -3000.0, 2000.0
    where(x)
    q, t = fp8.quantize(x, f8, square=square, both=True)
    check_held(q, x, f8, square)
    check_held(t, x.t(), f8, square)


def poisoned(M, N, K, seed):
    """Operands with NaN and infinities in some rows, and which results they reach."""
    x, w = matrix(M, K, seed, spread=0.3), matrix(N, K, seed + 1, spread=0.3)
    bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
    for i, v in ((0, math.nan), (M // 2, math.inf), (M - 1, -math.inf)):
        x[i, (7 * i) % K], bad[i] = v, True
    for j, v in ((N // 3, math.nan), (N - 1, math.inf)):
        w[j, (5 * j) % K], bad[:, j] = v, True
    return x, w, bad


# tiles of one SM of every width, split and whole; pairs of every width, rows in whole pieces and not, several tiles for a pair
@pytest.mark.parametrize("M,N,K", [(16, 136, 512), (17, 128, 640), (33, 1000, 1024), (64, 300, 130), (40, 1000, 4096), (1000, 40, 4096), (2656, 136, 730), (524, 4968, 644), (519, 5680, 632),
                                   (2306, 5576, 603), (5054, 129, 628), (2049, 4681, 604), (2561, 4993, 670)])
def test_products_of_values_that_are_not_finite(M, N, K):
    x, w, bad = poisoned(M, N, K, 1)
    for dtype in (torch.float16, torch.float32):
        got = fp8.matmul(fp8.quantize(x), fp8.quantize(w), dtype=dtype)
        assert torch.equal(got.isnan(), bad)                    # e4m3 holds an infinity as NaN
    # e5m2 holds it as one: each sum as 64 bits have it
    a, b = fp8.quantize(x, E5M2), fp8.quantize(w, E5M2)
    got, xv, wv = fp8.matmul(a, b, dtype=torch.float32), a.dequantize().double(), b.dequantize().double()
    assert bool(got[~bad].isfinite().all())
    sums = [(got[i], (xv[i] * wv).sum(1)) for i in (0, M // 2, M - 1)] + [(got[:, j], (xv * wv[j]).sum(1)) for j in (N // 3, N - 1)]
    for have, want in sums:
        kinds = lambda t: torch.where(t.isfinite(), 0.0, t.double()).nan_to_num(nan=2.0, posinf=1.0, neginf=-1.0)
        assert torch.equal(kinds(have), kinds(want))
    assert fp8.device_status() == 0


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", [40, 300, 1031])
def test_scales_that_are_not_a_number(dtype, cols):
    """float8_e8m0fnu has a NaN: a block with that scale has no value, and no product of it has one."""
    x = matrix(20, cols, 1, spread=0.3)
    x[3, 5] = 0
    q, w = fp8.quantize(x), fp8.quantize(matrix(136, cols, 2, spread=0.3))
    want = q.dequantize(TYPES[dtype])
    codes = q.scales.view(torch.uint8)
    codes[0, 3, 0] = 255
    want[3, :128] = math.nan
    got = q.dequantize(TYPES[dtype])
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    rows = fp8.matmul(q, w, dtype=torch.float32).isnan()
    assert bool(rows[3].all()) and int(rows.sum()) == 136


@pytest.mark.parametrize("f8", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", [256, 255])
def test_every_value_with_every_scale(f8, dtype, cols):
    """All 8-bit values in blocks of all scales, those of denormals and of values past fp32's range among them: rounded to fp32, then to the result's type."""
    data = torch.arange(256, dtype=torch.uint8, device="cuda")[:cols].repeat(256, 1)
    padded = torch.zeros((256, 256), dtype=torch.uint8, device="cuda")
    padded[:, :cols] = data
    codes = torch.zeros((1, 256, 4), dtype=torch.uint8, device="cuda")
    codes[0, :, 0] = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes[0, :, 1] = torch.arange(255, -1, -1, dtype=torch.uint8, device="cuda")
    got = fp8.BlockFp8(padded.view(f8)[:, :cols], codes.view(torch.float8_e8m0fnu)).dequantize(TYPES[dtype])
    scales = torch.where(codes[0, :, :2] == 255, math.nan, pow2(codes[0, :, :2].double() - 127)).repeat_interleave(128, 1)[:, :cols]
    want = (data.view(f8).double() * scales).float().to(TYPES[dtype])
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


# ---- frozen layers and their buffers ----

def frozen(cin=200, cout=131, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Linear(cin, cout).half().cuda()


def test_a_frozen_layer_multiplies_with_the_buffers_that_it_has():
    """Values or scales replaced alone, by assignment, from a file, or written in place, count in the next call."""
    x = matrix(30, 200, 1, torch.float16)
    a, b = fp8.Fp8Linear(frozen(seed=1)), fp8.Fp8Linear(frozen(seed=2))
    mlp = fp8.Fp8Mlp(frozen(seed=1), frozen(131, 72, 3))
    y, z = a(x), mlp(x)
    a.weight_scales = a.weight_scales + 1                                              # every scale twice as large
    assert torch.equal(a(x), fp8.matmul(fp8.quantize(x), fp8.quantize(2 * frozen(seed=1).weight, square=True), a.bias))
    a.weight_scales = a.weight_scales - 1
    assert torch.equal(a(x), y)
    a.load_state_dict({"weight_scales": a.weight_scales + 1}, strict=False, assign=True)
    assert not torch.equal(a(x), y)
    a.load_state_dict({"weight_scales": a.weight_scales - 1}, strict=False)
    assert torch.equal(a(x), y)
    a.weight_data, a.weight_scales, a.bias = b.weight_data, b.weight_scales, b.bias
    assert torch.equal(a(x), b(x))
    mlp.proj_scales.add_(1)
    assert not torch.equal(mlp(x), z)
    mlp.proj_scales = mlp.proj_scales - 1
    assert torch.equal(mlp(x), z)
    with pytest.raises(capi.VenomError, match="scales"):
        b.weight_scales = b.weight_scales[:, :-1]
        b(x)
    with pytest.raises(capi.VenomError, match="values"):
        mlp.fc_data = mlp.fc_data[:, :192]
        mlp(x)


def test_a_frozen_layer_that_leaves_the_device_leaves_its_memory():
    x = matrix(16, 2048, 1, torch.float16)
    layer = fp8.Fp8Linear(torch.nn.Linear(2048, 4096).half().cuda())
    layer(x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    layer.cpu()
    assert before - torch.cuda.memory_allocated() >= 2048 * 4096
    with pytest.raises(capi.VenomError, match="CUDA device"):
        layer(x)
    assert layer.cuda()(x).shape == (16, 4096)


@pytest.mark.parametrize("cin", [8, 24, 200, 208, 513])
def test_one_weight_always_gives_the_same_bytes(cin):
    lin = frozen(cin)
    states = []
    for fill in (0x5A, 0xC3):
        room = [torch.full((n,), fill, dtype=torch.uint8, device="cuda") for n in (1 << 18, 1 << 19, 1 << 20)]       # what the allocator hands out next
        del room
        states.append(fp8.Fp8Linear(lin).state_dict())
    assert states[0].keys() == states[1].keys()
    for k, v in states[0].items():
        assert torch.equal(v, states[1][k]), k
        assert v.untyped_storage().nbytes() == v.numel() * v.element_size(), k
    storages = {v.untyped_storage().data_ptr() for v in states[0].values()}
    assert len(storages) == len(states[0])


def test_frozen_layers_take_inputs_of_any_shape():
    lin, mlp = fp8.Fp8Linear(frozen()), fp8.Fp8Mlp(frozen(), frozen(131, 72))
    x = matrix(12, 200, 1, torch.float16)
    wide = torch.zeros(12, 207, dtype=torch.float16, device="cuda")
    wide[:, 5:205] = x
    for layer, out in ((lin, 131), (mlp, 72)):
        y = layer(x)
        assert torch.equal(layer(x.reshape(2, 3, 2, 200)), y.reshape(2, 3, 2, out)) and torch.equal(layer(x[0]), y[0]) and torch.equal(layer(wide[:, 5:205]), y)
        assert layer(x[:0]).shape == (0, out) and layer(x.reshape(2, 6, 200)[:, :0]).shape == (2, 0, out) and torch.equal(layer(x.t().contiguous().t()), y)
        for bad, match in ((x[:, :199], "do not match"), (x.cpu(), "CUDA"), (x.double(), "expected"), (x.sum(), "dimension"), (None, None)):
            with pytest.raises(capi.VenomError, match=match):
                layer(bad)


def test_a_layer_from_a_file_with_views():
    x, layer = matrix(30, 200, 1, torch.float16), fp8.Fp8Linear(frozen())
    state = layer.__dict__.copy()
    state["_views"] = {name: (cols, None, None) for name, cols in state.pop("_cols").items()}
    old = fp8.Fp8Linear.__new__(fp8.Fp8Linear)
    old.__setstate__(state)
    assert torch.equal(old(x), layer(x))


# ---- what is kept between the passes ----

def leaf(t):
    return t.detach().clone().requires_grad_()


def requested():
    """Bytes asked for and not freed yet; what the allocator rounds them up to depends on what it has at hand."""
    torch.cuda.synchronize()
    return torch.cuda.memory_stats()["requested_bytes.all.current"]


def bytes_kept(call, of):
    """Device memory that a graph holds besides its result, the leaves and their like."""
    start = requested()
    x = of * 1.0                                       # an input that lives only as long as the graph wants it
    y = call(x)
    del x
    kept = requested() - start - y.numel() * y.element_size()
    y.backward(torch.ones_like(y))
    return kept


ROOM = 1 << 16                                         # padding and scales of few rows


@pytest.mark.parametrize("tokens,cin,cout", [(256, 2048, 4096), (64, 1024, 4096), (4096, 1024, 1024), (1024, 4096, 1024), (1023, 2048, 1024), (2048, 4096, 4096)])
def test_a_linear_keeps_no_more_than_in_16_bits(tokens, cin, cout):
    x, w, b = leaf(matrix(tokens, cin, 1, torch.float16)), leaf(matrix(cout, cin, 2, torch.float16)), leaf(matrix(1, cout, 3, torch.float16)[0])
    kept, dense = bytes_kept(lambda t: fp8.linear(t, w, b), x), bytes_kept(lambda t: torch.nn.functional.linear(t, w, b), x)
    assert kept <= (cin * tokens + (cin * cout if cout <= tokens else 0)) * 129 / 128 + ROOM
    assert kept <= dense + ROOM and dense >= 2 * cin * tokens


def test_a_linear_with_32_bit_weights_keeps_no_more_than_a_cast_one():
    x, w = leaf(matrix(256, 1024, 1, torch.float16)), leaf(matrix(2048, 1024, 2))
    kept, dense = bytes_kept(lambda t: fp8.linear(t, w), x), bytes_kept(lambda t: torch.nn.functional.linear(t, w.half()), x)
    assert kept <= 1024 * (256 + 2048) * 129 / 128 + ROOM and 2 * kept <= dense + 2 * ROOM


@pytest.mark.parametrize("tokens,cin,hidden", [(256, 1024, 4096), (2048, 1024, 4096), (8192, 512, 2048)])
def test_a_feed_forward_block_keeps_no_more_than_in_16_bits(tokens, cin, hidden):
    x, w1, w2 = leaf(matrix(tokens, cin, 1, torch.float16)), leaf(matrix(hidden, cin, 2, torch.float16)), leaf(matrix(cin, hidden, 3, torch.float16))
    kept = bytes_kept(lambda t: fp8.mlp(t, w1, None, w2, None), x)
    dense = bytes_kept(lambda t: torch.nn.functional.linear(torch.nn.functional.gelu(torch.nn.functional.linear(t, w1)), w2), x)
    weights = sum(cin * hidden for rows in (hidden, cin) if rows <= tokens)
    assert kept <= (tokens * (cin + 2 * hidden) + weights) * 129 / 128 + ROOM and kept <= dense + ROOM


@pytest.mark.parametrize("tokens,cin,hidden,cout", [(37, 100, 203, 70), (37, 128, 33, 300), (1, 64, 128, 64), (300, 200, 515, 130), (0, 64, 128, 32)])
@pytest.mark.parametrize("w_type", ["fp16", "fp32"])
def test_gradients_are_the_same_whatever_is_kept_of_a_weight(tokens, cin, hidden, cout, w_type):
    """A leaf, and a weight that some operation made, whose transpose is kept."""
    t, dy = TYPES[w_type], matrix(tokens, cout, 9, torch.float16)
    x, w1, w2 = leaf(matrix(tokens, cin, 1, torch.float16)), leaf(matrix(hidden, cin, 2, t, 0.2)), leaf(matrix(cout, hidden, 3, t, 0.2))
    made = lambda w: w * 1.0
    a = torch.autograd.grad(fp8.mlp(x, w1, None, w2, None), (x, w1, w2), dy)
    b = torch.autograd.grad(fp8.mlp(x, made(w1), None, made(w2), None), (x, w1, w2), dy)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    w, dh = w1, matrix(tokens, hidden, 8, torch.float16)
    y = fp8.linear(x, w)
    a, again = torch.autograd.grad(y, (x, w), dh, retain_graph=True), torch.autograd.grad(y, (x, w), dh)
    b = torch.autograd.grad(fp8.linear(x, made(w)), (x, w), dh)
    only = torch.autograd.grad(fp8.linear(x, w.detach()), x, dh)[0]
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(a, b, again)) and torch.equal(only, a[0])


def test_a_weight_that_was_written_to_is_refused_or_kept():
    """Never a gradient of another weight than the forward pass's: few tokens keep the leaf, which torch refuses to use once it was written to; many keep its 8 bits."""
    for tokens, refused in ((40, True), (72, False), (200, False)):
        x, w, dy = leaf(matrix(tokens, 96, 1, torch.float16)), leaf(matrix(72, 96, 2, torch.float16)), matrix(tokens, 72, 3, torch.float16)
        (want,) = torch.autograd.grad(fp8.linear(x, w), x, dy)
        y = fp8.linear(x, w)
        with torch.no_grad():
            w.mul_(2)
        if refused:
            with pytest.raises(RuntimeError, match="inplace"):
                y.backward(dy)
        else:
            y.backward(dy)
            assert torch.equal(x.grad, want)


def test_saved_weights_in_another_form_are_refused():
    x, w = leaf(matrix(37, 100, 1, torch.float16)), leaf(matrix(70, 100, 2, torch.float16))
    for back in (lambda t: t[:-1] if t.dim() == 2 else t, lambda t: t.cpu() if t.dim() == 2 else t, lambda t: t.double() if t.dim() == 2 else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            y = fp8.linear(x, w)
        with pytest.raises(RuntimeError, match="another form"):
            y.backward(torch.ones_like(y))


def test_weights_made_in_inference_mode():
    with torch.inference_mode():
        w1, w2 = matrix(200, 96, 2, torch.float16), matrix(72, 200, 3, torch.float16)
    x, dy = leaf(matrix(16, 96, 1, torch.float16)), matrix(16, 72, 9, torch.float16)
    got = torch.autograd.grad(fp8.mlp(x, w1, None, w2, None), x, dy)[0]
    assert torch.equal(got, torch.autograd.grad(fp8.mlp(x, w1.clone(), None, w2.clone(), None), x, dy)[0])


# ---- models of several kinds of layers ----

def relative(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def test_attention_and_encoder_layers_convert():
    """Frozen linears inside modules that read their children's weights.  Operands in 8 bits are off by 2^-4 at most and 2^-5.8 of a standard deviation on average; two of them in
    each of two linears behind one another, whose result joins a residual stream of its size at least: 2^-5.8 * 2 = 2^-4.8 of it."""
    x = matrix(2 * 40, 64, 1, torch.float16, 0.0).reshape(2, 40, 64)
    torch.manual_seed(4)
    with torch.no_grad():
        attention = torch.nn.MultiheadAttention(64, 4, batch_first=True).half().cuda().eval()
        want = attention(x, x, x, need_weights=False)[0]
        assert torch.equal(fp8.linear_to_fp8(attention)(x, x, x, need_weights=False)[0], want)
        layer = torch.nn.TransformerEncoderLayer(64, 4, 256, dropout=0.0, activation="gelu", batch_first=True).half().cuda().eval()
        for model in (layer, torch.nn.TransformerEncoder(layer, 2, enable_nested_tensor=False)):
            want = model(x)
            for trainable in (True, False):
                got = fp8.linear_to_fp8(copy.deepcopy(model), trainable=trainable)(x)
                assert 0 < relative(got, want) <= 2.0 ** -4.8 * (2 if model is not layer else 1)


@pytest.mark.parametrize("pruned_first", [True, False])
def test_some_linears_pruned_and_the_rest_in_8_bits(pruned_first):
    """What linear_to_spmm skips becomes 8 bits, in either order; each layer computes what it computes alone."""
    from venom_b200 import nmv
    torch.manual_seed(5)
    net = torch.nn.ModuleDict({"query": torch.nn.Linear(256, 256), "out": torch.nn.Linear(256, 128), "ffn": torch.nn.Sequential(torch.nn.Linear(128, 512), torch.nn.GELU(), torch.nn.Linear(512, 128))})
    net = net.half().cuda().requires_grad_(False)
    dense = copy.deepcopy(net)
    steps = [lambda: nmv.linear_to_spmm(net, v=64, m=8, skip=("out", "ffn")), lambda: fp8.linear_to_fp8(net, skip=("query",))]
    for step in steps if pruned_first else steps[::-1]:
        step()
    assert type(net["query"]) is nmv.SrnmSpmm and all(type(m) is fp8.Fp8Linear for m in (net["out"], net["ffn"][0], net["ffn"][2]))
    x = matrix(72, 256, 1, torch.float16)
    h = net["query"](x)
    assert torch.equal(h, nmv.SrnmSpmm(dense["query"], v=64, m=8)(x))
    y = net["out"](h)
    assert torch.equal(y, fp8.linear(h, dense["out"].weight, dense["out"].bias))
    z = fp8.linear(torch.nn.functional.gelu(fp8.linear(y, dense["ffn"][0].weight, dense["ffn"][0].bias)), dense["ffn"][2].weight, dense["ffn"][2].bias)
    assert torch.equal(net["ffn"](y), z)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("trainable", [False, True])
def test_modules_under_autocast(dtype, trainable):
    """Results of the type that torch.nn.Linear gives there, those of the input in that type; gradients of the types of what they belong to."""
    t = TYPES[dtype]
    torch.manual_seed(6)
    fc, proj = torch.nn.Linear(96, 200).cuda(), torch.nn.Linear(200, 72).cuda()
    x, dy = matrix(50, 96, 1), matrix(50, 72, 2, t)
    for module, own in ((fp8.Fp8Linear(fc, trainable), lambda v: fp8.linear(v, fc.weight, fc.bias)), (fp8.Fp8Mlp(fc, proj, trainable=trainable), lambda v: fp8.mlp(v, fc.weight, fc.bias, proj.weight, proj.bias))):
        assert module(x).dtype == torch.float32
        with torch.autocast("cuda", dtype=t):
            y, dense = module(x), fc(x)
            with torch.autocast("cuda", enabled=False):
                assert module(x).dtype == torch.float32
            assert module(x.to(torch.bfloat16)).dtype == fc(x.to(torch.bfloat16)).dtype == t
        assert y.dtype == dense.dtype == t and torch.equal(y, own(x.to(t)))
    if trainable:
        v = leaf(x)
        with torch.autocast("cuda", dtype=t):
            y = module(v)
        y.backward(dy)
        assert v.grad.dtype == torch.float32 and fc.weight.grad.dtype == torch.float32
        (want,) = torch.autograd.grad(own(v.to(t)), v, dy)
        assert torch.equal(v.grad, want)
