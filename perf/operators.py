"""The block-scaled 8-bit operators as a list of measurable cases, with their plain forms.

  quantize  fp8.quantize(x): e4m3 or e5m2 values with a power of two for each block of 128 along a row (or of 128 x 128), and, where
            asked for, those of the transpose from the same pass
  matmul    fp8.matmul(a, b): a b^T of two such operands, sums in 32 bits
  linear    fp8.linear(x, w, bias) and its backward pass: the activation is kept as its 8-bit transpose until the weight's gradient is made
  gelu      fp8.gelu(x) and its backward pass from an 8-bit checkpoint of x
  mlp       fp8.mlp(x, w1, b1, w2, b2) and its backward pass: linear, GELU and linear, every kept activation in 8 bits

A block's scale is the smallest power of two s with amax / s <= the type's largest value (448 or 57344), where amax is the block's largest finite
magnitude; at least 2^-127.  Values are x / s rounded to nearest even.  Scales lie as [ceil(blocks / 4), rows, 4], blocks of four side by side.
"""
import math

import torch

own = False

E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
F8 = {"e4m3": E4M3, "e5m2": E5M2}


def listed():
    return [
        # the activations of one decoding step of sixteen sequences, ahead of the widest projection of a GPT-3-shaped block
        dict(name="quantize-decode", kind="quantize", rows=16, cols=12288, type="fp16", f8="e4m3", square=False, both=False),
        # a weight of that block made ready for training: itself and its transpose, one scale for 128 x 128 values
        dict(name="quantize-weight", kind="quantize", rows=12288, cols=12288, type="fp16", f8="e4m3", square=True, both=True),
        # one decoding step of a small model, where latency is all: BERT-large's square projections
        dict(name="matmul-small", kind="matmul", M=8, N=1024, K=1024, a="e4m3", b="e4m3", out="fp16", bias=True),
        # one decoding step through the widest projection of a GPT-3-shaped block: the weight's bytes are all
        dict(name="matmul-decode", kind="matmul", M=16, N=36864, K=12288, a="e4m3", b="e4m3", out="fp16", bias=True),
        # BERT-large's first feed-forward layer, batch 32 x sequence 512: few k for a tile
        dict(name="matmul-bert", kind="matmul", M=16384, N=4096, K=1024, a="e4m3", b="e4m3", out="fp16", bias=True),
        # an input gradient of a GPT-3-shaped block, one sequence of 2048 tokens; gradients in e5m2
        dict(name="matmul-gpt", kind="matmul", M=2048, N=12288, K=12288, a="e5m2", b="e4m3", out="bf16", bias=False),
        # a training step through BERT-large's first feed-forward layer
        dict(name="linear-bert", kind="linear", tokens=16384, cin=1024, cout=4096, type="fp16", weight="fp16", bias=True),
        # no round number, fp32 weights, no bias
        dict(name="linear-ragged", kind="linear", tokens=1371, cin=2039, cout=2978, type="bf16", weight="fp32", bias=False),
        # the activation between BERT-large's feed-forward layers
        dict(name="gelu-bert", kind="gelu", rows=16384, cols=4096, type="fp16", tanh=False),
        # ragged rows, the tanh form
        dict(name="gelu-ragged", kind="gelu", rows=1371, cols=2978, type="bf16", tanh=True),
        # a training step through BERT-large's feed-forward block, batch 16 x sequence 512
        dict(name="mlp-bert", kind="mlp", tokens=8192, hidden=1024, ffn=4096, type="fp16", bias=True, tanh=False),
        # a small ragged block, where launches count
        dict(name="mlp-ragged", kind="mlp", tokens=333, hidden=776, ffn=1537, type="bf16", bias=True, tanh=True),
    ]


MOST_FLOPS = 6.2e11
MOST_WEIGHT = 36864 * 12288


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "quantize", "matmul", "matmul", "matmul", "linear", "linear", "gelu", "mlp"])
    t = rng.choice(["fp16", "bf16"])
    while True:
        if kind == "quantize":
            c = dict(kind=kind, rows=_log(rng, 1, 36864), cols=_log(rng, 1, 12288), type=rng.choice(["fp16", "bf16", "fp32"]), f8=rng.choice(["e4m3", "e5m2"]),
                     square=rng.random() < 0.3, both=rng.random() < 0.6)
            fits = c["rows"] * c["cols"] <= 12288 * 12288
        elif kind == "matmul":
            c = dict(kind=kind, M=_log(rng, 1, 16384), N=_log(rng, 8, 36864), K=_log(rng, 16, 12288), a=rng.choice(["e4m3", "e4m3", "e5m2"]), b="e4m3",
                     out=rng.choice(["fp16", "bf16", "fp32"]), bias=rng.random() < 0.5)
            fits = c["N"] * c["K"] <= MOST_WEIGHT
        elif kind == "linear":
            c = dict(kind=kind, tokens=_log(rng, 1, 16384), cin=_log(rng, 64, 12288), cout=_log(rng, 64, 12288), type=t, weight=rng.choice([t, t, "fp32"]), bias=rng.random() < 0.6)
            fits = c["cin"] * c["cout"] <= 12288 * 4096
        elif kind == "gelu":
            c = dict(kind=kind, rows=_log(rng, 1, 16384), cols=_log(rng, 16, 12288), type=t, tanh=rng.random() < 0.5)
            fits = c["rows"] * c["cols"] <= 16384 * 4096
        else:
            c = dict(kind=kind, tokens=_log(rng, 16, 8192), hidden=_log(rng, 64, 2048), ffn=_log(rng, 128, 8192), type=t, bias=rng.random() < 0.7, tanh=rng.random() < 0.5)
            fits = True
        if fits and work(c)["flops"] <= MOST_FLOPS:
            return c


def work(case):
    c, kind = case, case["kind"]
    size = {"fp16": 2, "bf16": 2, "fp32": 4}

    def packed(rows, cols):
        return rows * cols + rows * -(-cols // 128)

    if kind == "quantize":
        out = packed(c["rows"], c["cols"]) + (packed(c["cols"], c["rows"]) if c["both"] else 0)
        return {"bytes": size[c["type"]] * c["rows"] * c["cols"] + out, "flops": 0.0}
    if kind == "matmul":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": packed(M, K) + packed(N, K) + size[c["out"]] * M * N + (2 * N if c["bias"] else 0), "flops": 2.0 * M * N * K}
    if kind == "linear":
        T, I, O = c["tokens"], c["cin"], c["cout"]
        # x, dy, w and the 8-bit checkpoint read, y, dx, dw and the checkpoint written
        return {"bytes": 2 * size[c["type"]] * T * (I + O) + 2 * size[c["weight"]] * I * O + 2 * T * I, "flops": 6.0 * T * I * O}
    if kind == "gelu":
        # x and dy read, y and dx written, the checkpoint both
        return {"bytes": c["rows"] * c["cols"] * (4 * size[c["type"]] + 2), "flops": 0.0}
    T, H, F = c["tokens"], c["hidden"], c["ffn"]
    # x, dy, y, dx and the weights with their gradients; checkpoints of x, of the first product and of its GELU
    return {"bytes": 4 * size[c["type"]] * T * H + 4 * size[c["type"]] * H * F + 2 * T * (H + 2 * F), "flops": 12.0 * T * H * F}


# ---------------------------------------------------------------------------------------------------------------------
# inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activation(rows, cols, g, dtype):
    """Normal values with channels of different size, as a layer's input has them."""
    x = torch.randn((rows, cols), device="cuda", generator=g)
    x *= torch.exp(0.7 * torch.randn((1, cols), device="cuda", generator=g))
    return x.to(dtype)


def _gradient(rows, cols, g, dtype):
    """Small values whose size differs from token to token."""
    x = torch.randn((rows, cols), device="cuda", generator=g)
    x *= 2e-3 * torch.exp(torch.randn((rows, 1), device="cuda", generator=g))
    return x.to(dtype)


def _weight(rows, cols, g, dtype):
    return (0.02 * torch.randn((rows, cols), device="cuda", generator=g)).to(dtype)


def _padded(data):
    """The same values in rows whose stride is a multiple of 16 bytes."""
    rows, cols = data.shape
    store = torch.zeros((rows, -(-cols // 16) * 16), dtype=torch.uint8, device=data.device)
    store[:, :cols] = data.view(torch.uint8)
    return store.view(data.dtype)[:, :cols]


def prepare(case, seed):
    c, kind, g = case, case["kind"], _generator(seed)
    s = dict(case=c)
    if kind == "quantize":
        make = _weight if c["square"] else _gradient if c["f8"] == "e5m2" else _activation
        s["x"] = make(c["rows"], c["cols"], g, TYPES[c["type"]])
    elif kind == "matmul":
        make = _gradient if c["a"] == "e5m2" else _activation
        data, s["sa"] = _quantize(make(c["M"], c["K"], g, torch.float32), F8[c["a"]], False)
        s["a"] = _padded(data)
        data, s["sb"] = _quantize(_weight(c["N"], c["K"], g, torch.float32), F8[c["b"]], True)
        s["b"] = _padded(data)
        s["bias"] = _weight(1, c["N"], g, torch.float16 if c["out"] == "fp32" else TYPES[c["out"]])[0] if c["bias"] else None
    elif kind == "linear":
        t, w = TYPES[c["type"]], TYPES[c["weight"]]
        s["x"] = _activation(c["tokens"], c["cin"], g, t).requires_grad_()
        s["w"] = _weight(c["cout"], c["cin"], g, w).requires_grad_()
        s["bias"] = _weight(1, c["cout"], g, w)[0].requires_grad_() if c["bias"] else None
        s["dy"] = _gradient(c["tokens"], c["cout"], g, t)
    elif kind == "gelu":
        t = TYPES[c["type"]]
        s["x"] = _activation(c["rows"], c["cols"], g, t).requires_grad_()
        s["dy"] = _gradient(c["rows"], c["cols"], g, t)
    elif kind == "mlp":
        t, T, H, F = TYPES[c["type"]], c["tokens"], c["hidden"], c["ffn"]
        s["x"] = _activation(T, H, g, t).requires_grad_()
        s["w1"], s["w2"] = _weight(F, H, g, t).requires_grad_(), _weight(H, F, g, t).requires_grad_()
        s["b1"], s["b2"] = (_weight(1, F, g, t)[0].requires_grad_(), _weight(1, H, g, t)[0].requires_grad_()) if c["bias"] else (None, None)
        s["dy"] = _gradient(T, H, g, t)
    else:
        raise ValueError("unknown kind %r" % kind)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms


def _blocks(x, rows, cols):
    """x padded with zeros to whole blocks: [row blocks, rows, column blocks, cols]."""
    r, c = -(-x.shape[0] // rows), -(-x.shape[1] // cols)
    x = torch.nn.functional.pad(x, (0, c * cols - x.shape[1], 0, r * rows - x.shape[0]))
    return x.reshape(r, rows, c, cols)


def _quantize(x, f8, square):
    """(values [rows, cols] in 8 bits, scales [ceil(blocks / 4), rows, 4])."""
    n, k = x.shape
    b = _blocks(x.float(), 128 if square else 1, 128)
    m = b.abs()
    amax = torch.where(torch.isfinite(m), m, torch.zeros_like(m)).amax((1, 3))
    mant, exp = torch.frexp(amax)                                    # amax = mant 2^exp, mant in [0.5, 1)
    exp = exp - 1 - (8 if f8 == E4M3 else 15) + (mant > 0.875).int()  # the largest value is 1.75 2^8 or 1.75 2^15
    exp = torch.where(amax > 0, exp, torch.full_like(exp, -127)).clamp(min=-127)
    scaled = torch.ldexp(b, -exp[:, None, :, None])
    data = scaled.reshape(b.shape[0] * b.shape[1], -1)[:n, :k].to(f8)
    code = (exp + 127).to(torch.uint8).repeat_interleave(128 if square else 1, 0)[:n]
    groups = -(-code.shape[1] // 4)
    code = torch.nn.functional.pad(code, (0, 4 * groups - code.shape[1]))
    return data, code.reshape(n, groups, 4).transpose(0, 1).contiguous().view(E8M0)


def _values(data, scales):
    """What the 8-bit values stand for, in 32 bits."""
    n, k = data.shape
    s = scales.float().transpose(0, 1).reshape(n, -1)
    return data.float() * s.repeat_interleave(128, 1)[:, :k]


def _held(x, f8=E4M3, square=False):
    """x in 32 bits as its 8-bit form holds it."""
    return _values(*_quantize(x, f8, square))


def _gelu(x, tanh):
    """(GELU of x, its derivative) in 32 bits."""
    if tanh:
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)
    cdf = 0.5 * torch.erfc(x * -math.sqrt(0.5))
    return x * cdf, cdf + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))


def _plain_linear(s):
    c, x, w, dy = s["case"], s["x"].detach(), s["w"].detach(), s["dy"]
    hw = _held(w, square=True)
    y = _held(x) @ hw.T
    if s["bias"] is not None:
        y += s["bias"].detach().float()
    dx = _held(dy) @ hw
    dw = _held(dy.T) @ _held(x.T).T
    t, tw = TYPES[c["type"]], TYPES[c["weight"]]
    out = {"y": y.to(t), "dx": dx.to(t), "dw": dw.to(tw)}
    if s["bias"] is not None:
        out["db"] = dy.float().sum(0).to(tw)
    return out


def _plain_mlp(s):
    c, x, dy = s["case"], s["x"].detach(), s["dy"]
    t, tanh = TYPES[c["type"]], c["tanh"]
    h1, h2 = _held(s["w1"].detach(), square=True), _held(s["w2"].detach(), square=True)
    h = _held(x) @ h1.T
    if s["b1"] is not None:
        h += s["b1"].detach().float()
    h = h.to(t).float()
    act = _gelu(h, tanh)[0]
    y = _held(act) @ h2.T
    if s["b2"] is not None:
        y += s["b2"].detach().float()
    da = (_held(dy) @ h2).to(t).float()
    dh = da * _gelu(_held(h), tanh)[1]
    out = {"y": y.to(t), "dx": (_held(dh) @ h1).to(t), "dw1": (_held(dh.T) @ _held(x.T).T).to(t), "dw2": (_held(dy.T) @ _held(act.T).T).to(t)}
    if s["b1"] is not None:
        out["db1"], out["db2"] = dh.sum(0).to(t), dy.float().sum(0).to(t)
    return out


def _plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "quantize":
        data, scales = _quantize(s["x"], F8[c["f8"]], c["square"])
        out = {"data": data, "scales": scales}
        if c["both"]:
            out["data_t"], out["scales_t"] = _quantize(s["x"].T, F8[c["f8"]], c["square"])
        return out
    if kind == "matmul":
        y = _values(s["a"], s["sa"]) @ _values(s["b"], s["sb"]).T
        if s["bias"] is not None:
            y += s["bias"].float()
        return y.to(TYPES[c["out"]])
    if kind == "linear":
        return _plain_linear(s)
    if kind == "gelu":
        t = TYPES[c["type"]]
        x = s["x"].detach()
        return {"y": _gelu(x.float(), c["tanh"])[0].to(t), "dx": (s["dy"].float() * _gelu(_held(x), c["tanh"])[1]).to(t)}
    return _plain_mlp(s)


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls


def _own(s):
    from venom_b200 import fp8

    c, kind = s["case"], s["case"]["kind"]
    if kind == "quantize":
        q = fp8.quantize(s["x"], F8[c["f8"]], square=c["square"], both=c["both"])
        if c["both"]:
            return {"data": q[0].data, "scales": q[0].scales, "data_t": q[1].data, "scales_t": q[1].scales}
        return {"data": q.data, "scales": q.scales}
    if kind == "matmul":
        return fp8.matmul(fp8.BlockFp8(s["a"], s["sa"]), fp8.BlockFp8(s["b"], s["sb"]), s["bias"], dtype=TYPES[c["out"]])
    if kind == "linear":
        y = fp8.linear(s["x"], s["w"], s["bias"])
        leaves = [s["x"], s["w"]] + ([s["bias"]] if s["bias"] is not None else [])
        return dict(zip(("y", "dx", "dw", "db"), [y] + list(torch.autograd.grad(y, leaves, s["dy"]))))
    if kind == "gelu":
        y = fp8.gelu(s["x"], approximate="tanh" if c["tanh"] else "none")
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    y = fp8.mlp(s["x"], s["w1"], s["b1"], s["w2"], s["b2"], approximate="tanh" if c["tanh"] else "none")
    names = [n for n in ("x", "w1", "w2", "b1", "b2") if s[n] is not None]
    return dict(zip(["y"] + ["d" + n for n in names], [y] + list(torch.autograd.grad(y, [s[n] for n in names], s["dy"]))))


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits


def _held64(x, f8="e4m3", square=False, parts=False):
    """The values that the 8-bit form of x stands for; with `parts` (values in units of their scale, scales)."""
    top, low, bits = (448.0, -6, 3) if f8 == "e4m3" else (57344.0, -14, 2)
    x = x.double()
    n, k = x.shape
    tall = 128 if square else 1
    nb, kb = -(-n // tall), -(-k // 128)
    full = x.new_zeros((nb * tall, kb * 128))
    full[:n, :k] = x
    b = full.view(nb, tall, kb, 128)
    amax = b.abs().nan_to_num(0, 0, 0).amax(dim=(1, 3), keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(amax / top)).clamp(min=-127))
    # the logarithm is rounded: one step up or down where the quotient is next to a power of two
    s = torch.where(amax / s > top, 2 * s, s)
    s = torch.where((amax / s <= top / 2) & (s > 2.0 ** -127), s / 2, s)
    v = b / s
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** low))) - bits)
    v = torch.round(v / step) * step
    if parts:
        return v.reshape(nb * tall, kb * 128)[:n, :k], s.expand(nb, tall, kb, 1).reshape(nb * tall, kb)[:n]
    return (v * s).reshape(nb * tall, kb * 128)[:n, :k]


def _gelu64(x, tanh):
    if tanh:
        u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        sig = torch.sigmoid(2 * u)                  # (1 + tanh u) / 2
        return x * sig, sig + x * sig * torch.sigmoid(-2 * u) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * x ** 2)
    cdf = torch.special.ndtr(x)
    return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


def _unpack64(data, scales):
    g, n, _ = scales.shape
    per_block = scales.double().permute(1, 0, 2).reshape(n, 4 * g)
    return data.double() * per_block.repeat_interleave(128, dim=1)[:, : data.shape[1]]


def exact(case, seed):
    c, kind, s = case, case["kind"], prepare(case, seed)

    def laid_out(x):
        v, sc = _held64(x, c["f8"], c["square"], parts=True)
        groups = -(-sc.shape[1] // 4)
        full = sc.new_full((sc.shape[0], 4 * groups), 2.0 ** -127)
        full[:, : sc.shape[1]] = sc
        return v, full.view(-1, groups, 4).permute(1, 0, 2)

    with torch.no_grad():
        if kind == "quantize":
            out = dict(zip(("data", "scales"), laid_out(s["x"])))
            if c["both"]:
                out.update(zip(("data_t", "scales_t"), laid_out(s["x"].t())))
            return out
        if kind == "matmul":
            y = _unpack64(s["a"], s["sa"]) @ _unpack64(s["b"], s["sb"]).t()
            return y if s["bias"] is None else y + s["bias"].double()
        if kind == "linear":
            w = _held64(s["w"], square=True)
            out = {"y": _held64(s["x"]) @ w.t(), "dx": _held64(s["dy"]) @ w, "dw": _held64(s["dy"].t()) @ _held64(s["x"].t()).t()}
            if s["bias"] is not None:
                out["y"] += s["bias"].double()
                out["db"] = s["dy"].double().sum(dim=0)
            return out
        if kind == "gelu":
            return {"y": _gelu64(s["x"].double(), c["tanh"])[0], "dx": s["dy"].double() * _gelu64(_held64(s["x"]), c["tanh"])[1]}
        t = TYPES[c["type"]]
        w1, w2 = _held64(s["w1"], square=True), _held64(s["w2"], square=True)
        h = _held64(s["x"]) @ w1.t()
        if s["b1"] is not None:
            h = h + s["b1"].double()
        h = h.to(t).double()                        # what is kept between the two halves has the activations' type, by definition
        act = _gelu64(h, c["tanh"])[0]
        y = _held64(act) @ w2.t()
        dh = (_held64(s["dy"]) @ w2).to(t).double() * _gelu64(_held64(h), c["tanh"])[1]
        out = {"y": y, "dx": _held64(dh) @ w1, "dw1": _held64(dh.t()) @ _held64(s["x"].t()).t(), "dw2": _held64(s["dy"].t()) @ _held64(act.t()).t()}
        if s["b1"] is not None:
            out["y"] = y + s["b2"].double()
            out["db1"], out["db2"] = dh.sum(dim=0), s["dy"].double().sum(dim=0)
        return out
