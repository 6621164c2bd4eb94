"""Cases of layer normalisation and of 8-bit activation checkpoints, in plain torch operations and through the package.

Operators (the "op" of a case):
  ln_forward   y = gamma (x - mean) rstd + beta per row, with mean and rstd; optionally the normalised rows kept in 8 bits
  ln_backward  dx, dgamma, dbeta, the normalised rows taken from x (mean, rstd) or from an 8-bit checkpoint
  checkpoint   a tensor stored in 8 bits and read back
  function     the error below a neuron function whose input was kept in 8 bits
  wgrad        the weight and bias gradient of a Linear layer whose input was kept in 8 bits

The 8-bit form: a row is cut into blocks of 32 values; a block has one exponent byte b and a signed byte q per value, which
stand for q/64 * 2^(b-127).  b is the exponent field of the block's largest magnitude, one more where that value would round
to 128; q is rounded to nearest, ties to even.
"""
import math

import torch

own = False

EPS = 1e-6
BLOCK = 32
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
FUNCTIONS = ("sigmoid", "tanh", "relu", "leaky_relu")
SLOPE = 0.1


def listed():
    return [
        # one latent vector of 256 values normalised when a single sample is answered: latency
        dict(name="ln_forward_latent", op="ln_forward", rows=1, n=256, type="float32", checkpoint=False),
        # a training batch of 128 samples of 32 x 64 x 64 normalised per sample, normalised values kept in 8 bits
        dict(name="ln_forward_sample", op="ln_forward", rows=128, n=131072, type="float32", checkpoint=True),
        # backward pass over the latent vectors of a batch: latency
        dict(name="ln_backward_latent", op="ln_backward", rows=128, n=256, type="float32", checkpoint=False),
        # many rows of an odd length in half precision
        dict(name="ln_backward_ragged", op="ln_backward", rows=5003, n=1021, type="float16", checkpoint=False),
        # 64 samples of 64 x 32 x 32 (first stage of a discriminator), normalised per sample: few long rows
        dict(name="ln_backward_sample", op="ln_backward", rows=64, n=65536, type="float32", checkpoint=False),
        # many feature rows, the forward pass kept 8 bits a value
        dict(name="ln_backward_8bit", op="ln_backward", rows=16384, n=2048, type="bfloat16", checkpoint=True),
        # ragged rows in half precision stored and read back
        dict(name="checkpoint_ragged", op="checkpoint", rows=509, n=4099, type="float16"),
        # the first activation of a batch of 128 images (32 x 128 x 128 a sample)
        dict(name="checkpoint_images", op="checkpoint", rows=128, n=524288, type="float32"),
        # the hidden layer of a small head
        dict(name="function_head", op="function", rows=64, n=1000, type="bfloat16", func="tanh"),
        # the function layer behind the first convolution of a batch of 128 images
        dict(name="function_images", op="function", rows=128, n=524288, type="float32", func="leaky_relu"),
        # weight gradient of a head on 256 x 8 x 8 features of a batch of 128: few rows, output bound
        dict(name="wgrad_head", op="wgrad", rows=128, n=16384, out=256, type="float32"),
        # weight gradient of a wide layer over many rows
        dict(name="wgrad_wide", op="wgrad", rows=8192, n=4096, out=4096, type="bfloat16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("ln_forward", "ln_backward", "checkpoint", "function", "wgrad"))
    case = dict(op=op, type=rng.choice(tuple(TYPES)))
    if op == "wgrad":
        case["rows"] = _spread(rng, 1, 16384)
        case["n"], case["out"] = _spread(rng, 8, 8192), _spread(rng, 1, 4096)
        while case["rows"] * case["n"] * case["out"] > 8192 * 4096 * 2048:
            case["rows"] = max(1, case["rows"] // 2)
        return case
    most = 1 << 24 if op in ("ln_forward", "ln_backward") else 1 << 25
    case["n"] = _spread(rng, 16, 262144)
    case["rows"] = _spread(rng, 1, min(32768, most // case["n"]))
    if op in ("ln_forward", "ln_backward"):
        case["checkpoint"] = rng.random() < 0.4
    if op == "function":
        case["func"] = rng.choice(FUNCTIONS)
    return case


# ---- the 8-bit form in elementary operations ------------------------------------------------------

def _blocks(x):
    rows, n = x.shape
    pad = -n % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).view(rows, -1, BLOCK)


def _encode(x):
    """codes [rows, 32 blocks] int8 and exponents [rows, blocks] uint8 of x [rows, n] in 32 bits (finite values)."""
    v = _blocks(x)
    top = v.abs().amax(2)
    b = (top.view(torch.int32) >> 23).clamp(min=1)
    # x / 2^(b-133) in two exact steps: the factor alone can leave the range of 32 bits
    up = torch.ldexp(torch.ones_like(top), 125 - b)
    b = b + ((top * up * 256 >= 127.5) & (b < 254)).to(torch.int32)
    up = torch.ldexp(torch.ones_like(top), 125 - b)
    q = torch.round(v * up.unsqueeze(2) * 256).clamp(-127, 127)
    return q.to(torch.int8).view(x.shape[0], -1), b.to(torch.uint8)


def _decode(codes, exponents, n):
    """The values in 32 bits, [rows, n]."""
    rows = codes.shape[0]
    scale = torch.ldexp(torch.ones(exponents.shape, device=codes.device), exponents.to(torch.int32) - 127)
    v = codes.view(rows, -1, BLOCK).to(torch.float32) / 64 * scale.unsqueeze(2)
    return v.view(rows, -1)[:, :n]


# ---- inputs -----------------------------------------------------------------------------------------

def _numbers(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *shape: torch.randn(*shape, device="cuda", generator=g)


def prepare(case, seed):
    rows, n, kind = case["rows"], case["n"], TYPES[case["type"]]
    normal = _numbers(case, seed)
    s = dict(case=case)
    if case["op"] == "ln_forward":
        s["x"] = (normal(rows, n) * (1 + 0.2 * normal(rows, 1)) + 0.5 + 0.3 * normal(rows, 1)).to(kind)
        s["gamma"], s["beta"] = 1 + 0.1 * normal(n), 0.1 * normal(n)
        s["y"], s["mean"], s["rstd"] = torch.empty_like(s["x"]), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        if case["checkpoint"]:
            s["codes"], s["exponents"] = _room(rows, n)
            s["kept"] = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    elif case["op"] == "ln_backward":
        x = (normal(rows, n) * (1 + 0.2 * normal(rows, 1)) + 0.5 + 0.3 * normal(rows, 1)).to(kind)
        s["dy"], s["gamma"] = normal(rows, n).to(kind), 1 + 0.1 * normal(n)
        mean = x.mean(1, dtype=torch.float64, keepdim=True)
        rstd = ((x - mean).square().mean(1, keepdim=True) + EPS).rsqrt()
        s["mean"], s["rstd"] = mean.float().view(-1), rstd.float().view(-1)
        if case["checkpoint"]:
            s["codes"], s["exponents"] = _encode(((x - mean) * rstd).float())
        else:
            s["x"] = x
        s["dx"], s["dgamma"], s["dbeta"] = torch.empty_like(s["dy"]), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    elif case["op"] == "checkpoint":
        s["x"] = (normal(rows, n) * torch.exp(0.5 * normal(rows, 1))).to(kind)
        s["codes"], s["exponents"] = _room(rows, n)
        s["out"] = torch.empty_like(s["x"])
    elif case["op"] == "function":
        s["codes"], s["exponents"] = _encode(1.5 * normal(rows, n))
        s["error"] = normal(rows, n).to(kind)
        s["out"] = torch.empty_like(s["error"])
    else:
        x = normal(rows, n)
        s["codes"], s["exponents"] = _encode(torch.where(x > 0, x, SLOPE * x))
        s["delta"] = (normal(rows, case["out"]) / math.sqrt(rows)).to(kind)
        s["dweight"], s["dbias"] = torch.empty(case["out"], n, device="cuda"), torch.empty(case["out"], device="cuda")
    return s


def _room(rows, n):
    blocks = -(-n // BLOCK)
    return (torch.empty(rows, blocks * BLOCK, dtype=torch.int8, device="cuda"),
            torch.empty(rows, blocks, dtype=torch.uint8, device="cuda"))


# ---- one pass ---------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return globals()["_plain_" + s["case"]["op"]](s)


def _run_own(s):
    from cuda_cnn_gan_vae_b200 import ops
    case = s["case"]
    op, n = case["op"], case["n"]
    kept = ops.Checkpoint8(s["codes"], s["exponents"], n) if "codes" in s else None
    if op == "ln_forward":
        ops.ln_forward(s["x"], s["gamma"], s["beta"], EPS, y=s["y"], mean=s["mean"], rstd=s["rstd"], checkpoint=kept)
        if kept is None:
            return [s["y"], s["mean"], s["rstd"]]
        kept.load(s["kept"])
        return [s["y"], s["mean"], s["rstd"], s["kept"]]
    if op == "ln_backward":
        ops.ln_backward(s["dy"], s["x"] if kept is None else kept, s["mean"], s["rstd"], s["gamma"], s["dgamma"], s["dbeta"],
                        accumulate=False, dx=s["dx"])
        return [s["dx"], s["dgamma"], s["dbeta"]]
    if op == "checkpoint":
        kept.store(s["x"])
        return kept.load(s["out"])
    if op == "function":
        ops.CTensorApplyFunc.Backward(s["out"], kept, s["error"], case["func"], SLOPE)
        return s["out"]
    ops.checkpoint_wgrad(s["dweight"], s["dbias"], s["delta"], kept, accumulate=False)
    return [s["dweight"], s["dbias"]]


def _plain_ln_forward(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt(c.square().mean(1, keepdim=True) + EPS)
    xhat = c * rstd
    out = [(xhat * s["gamma"] + s["beta"]).to(s["x"].dtype), mean.view(-1), rstd.view(-1)]
    if s["case"]["checkpoint"]:
        out.append(_decode(*_encode(xhat), s["case"]["n"]).to(torch.bfloat16))
    return out


def _plain_ln_backward(s):
    dy, rstd = s["dy"].float(), s["rstd"].view(-1, 1)
    if s["case"]["checkpoint"]:
        xhat = _decode(s["codes"], s["exponents"], s["case"]["n"])
    else:
        xhat = (s["x"].float() - s["mean"].view(-1, 1)) * rstd
    g = dy * s["gamma"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return [dx.to(s["dy"].dtype), (dy * xhat).sum(0), dy.sum(0)]


def _plain_checkpoint(s):
    return _decode(*_encode(s["x"].float()), s["case"]["n"]).to(s["x"].dtype)


def _plain_function(s):
    z, func = _decode(s["codes"], s["exponents"], s["case"]["n"]), s["case"]["func"]
    if func == "sigmoid":
        f = 1 / (1 + torch.exp(-z))
        slope = (1 - f) * f
    elif func == "tanh":
        slope = 1 - torch.tanh(z).square()
    else:
        slope = torch.where(z >= 0, 1.0, SLOPE if func == "leaky_relu" else 0.0)
    return (slope * s["error"].float()).to(s["error"].dtype)


def _plain_wgrad(s):
    delta = s["delta"].float()
    return [delta.t() @ _decode(s["codes"], s["exponents"], s["case"]["n"]), delta.sum(0)]


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    rows, n, size = case["rows"], case["n"], SIZE[case["type"]]
    values, kept = rows * n, rows * -(-n // BLOCK) * (BLOCK + 1)
    if case["op"] == "ln_forward":
        b = 2 * size * values + 8 * n + 8 * rows
        # what is kept is written and read back, its values come out in 16 bits
        return dict(bytes=b + (2 * kept + 2 * values if case["checkpoint"] else 0), flops=8 * values)
    if case["op"] == "ln_backward":
        b = 2 * size * values + 12 * n + 8 * rows
        return dict(bytes=b + (kept if case["checkpoint"] else size * values), flops=14 * values)
    if case["op"] == "checkpoint":
        return dict(bytes=2 * size * values + 2 * kept, flops=4 * values)
    if case["op"] == "function":
        return dict(bytes=2 * size * values + kept, flops=8 * values)
    out = case["out"]
    return dict(bytes=size * rows * out + kept + 4 * n * out + 4 * out, flops=2 * values * out)


# ---- the definitions in 64 bits ----------------------------------------------------------------------

def _held(v):
    """The values that the 8-bit form of v (64 bits, [rows, n]) stands for."""
    rows, n = v.shape
    wide = torch.zeros(rows, -(-n // 32) * 32, dtype=torch.float64, device=v.device)
    wide[:, :n] = v
    wide = wide.reshape(rows, -1, 32)
    largest = wide.abs().max(dim=2, keepdim=True).values
    # 2^power <= largest < 2^(power + 1)
    power = (torch.frexp(largest).exponent - 1).clamp(min=-126).double()
    step = torch.exp2(power - 6)
    step = torch.where((torch.round(largest / step) > 127) & (power < 127), 2 * step, step)
    held = torch.clamp(torch.round(wide / step), min=-127, max=127) * step
    return held.reshape(rows, -1)[:, :n]


def _stands_for(s):
    """What the codes and exponents of a state stand for, in 64 bits."""
    q = s["codes"].double()
    b = s["exponents"].double().repeat_interleave(32, dim=1)
    return (q * torch.exp2(b - 133))[:, :s["case"]["n"]]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "ln_forward":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        xhat = (x - mean) / (var + EPS).sqrt()
        y = torch.addcmul(s["beta"].double(), xhat, s["gamma"].double())
        got = [y, mean.flatten(), (var + EPS).pow(-0.5).flatten()]
        # the kept value is that of the normalised row
        return got + [_held(xhat)] if case["checkpoint"] else got
    if op == "ln_backward":
        dy, gamma = s["dy"].double(), s["gamma"].double()
        xhat = _stands_for(s) if case["checkpoint"] else (s["x"].double() - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
        n = case["n"]
        first = torch.mv(dy, gamma) / n
        second = torch.mv(dy * xhat, gamma) / n
        dx = (dy * gamma - first[:, None] - xhat * second[:, None]) * s["rstd"].double()[:, None]
        return [dx, torch.einsum("rn,rn->n", dy, xhat), dy.sum(dim=0)]
    if op == "checkpoint":
        return _held(s["x"].double())
    if op == "function":
        z, func = _stands_for(s), case["func"]
        if func == "sigmoid":
            d = 0.25 / torch.cosh(z / 2).square()
        elif func == "tanh":
            d = torch.cosh(z).pow(-2)
        else:
            d = torch.ones_like(z)
            d[z < 0] = SLOPE if func == "leaky_relu" else 0.0
        return d * s["error"].double()
    return [torch.matmul(s["delta"].double().t(), _stands_for(s)), s["delta"].double().sum(dim=0)]
