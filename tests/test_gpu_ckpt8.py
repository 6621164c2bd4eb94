"""8-bit activation checkpoints on the GPU: the format bit for bit, and their use in the backward pass against 64 bits."""
import numpy as np
import pytest
import torch

from tests import ckpt8_util as cu

pytestmark = pytest.mark.gpu
KINDS = ["float32", "bfloat16", "float16"]
SIZES = [(1, 1), (3, 31), (4, 32), (5, 33), (1, 100), (129, 64), (7, 1000), (33, 4099), (2, 100001), (1000, 96)]


@pytest.fixture(autouse=True)
def ops():
    from cuda_cnn_gan_vae_b200 import ops
    return ops


def spread(rows, n, kind, seed=0):
    """Values over the whole range of the type, block by block, with zeros, ties of the rounding and borders of the exponent."""
    r = np.random.default_rng(seed + rows * 31 + n)
    low, high = {"float32": (-149, 127), "bfloat16": (-133, 127), "float16": (-24, 15)}[kind]
    x = r.normal(0, 1, (rows, n)) * np.ldexp(1.0, np.repeat(r.integers(low, high - 1, (rows, -(-n // 32))), 32, axis=1)[:, :n])
    special = np.array([0.0, 127.5, 127.4999, 127.0, 0.5, 1.5, 2.5, -0.5, -126.5, 64.0, 63.5, 128.0, -0.0, 1e-3, -1e-3])
    pick = r.random((rows, n)) < 0.1
    x = np.where(pick, special[r.integers(0, len(special), (rows, n))], x)
    top = float(torch.finfo(getattr(torch, kind)).max)
    return torch.from_numpy(np.clip(x, -top, top)).to(getattr(torch, kind)).cuda()


def wide(x):
    return x.double().cpu().numpy()


@pytest.mark.parametrize("keep_sign", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", SIZES)
def test_format_bit_for_bit(ops, rows, n, kind, keep_sign):
    x = spread(rows, n, kind)
    c = ops.Checkpoint8.empty(rows, n)
    c.store(x, keep_sign=keep_sign)
    codes, exponents = cu.encode(wide(x), keep_sign)
    np.testing.assert_array_equal(c.exponents.cpu().numpy(), exponents)
    np.testing.assert_array_equal(c.codes.cpu().numpy(), codes)
    values = cu.decode(codes, exponents, n)
    for out in KINDS:
        t = getattr(torch, out)
        got = c.load(torch.empty(rows, n, dtype=t, device="cuda"))
        top = float(torch.finfo(t).max)
        want = torch.from_numpy(np.clip(values, -top, top)).to(t) if out == "float16" else torch.from_numpy(values).to(t)
        assert torch.equal(got.cpu(), want), out
        if out != "float16":
            np.testing.assert_array_equal(wide(got), values)          # 8 bits are exact in fp32 and bf16
    ops.stream_status()


def test_largest_and_smallest_numbers(ops):
    top = torch.finfo(torch.float32).max
    x = torch.zeros(5, 64, device="cuda")
    x[0, 5], x[0, 6] = top, -top                   # saturates at 127 steps instead of overflowing
    x[1, 40] = 2.0 ** -149                         # the smallest subnormal number
    x[2, :] = 2.0 ** -126
    x[3, 3], x[3, 4] = 2.0 ** 127 * 1.99, 1.0
    c = ops.Checkpoint8.empty(5, 64).store(x)
    codes, exponents = cu.encode(wide(x))
    np.testing.assert_array_equal(c.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(c.exponents.cpu().numpy(), exponents)
    got = wide(c.load(torch.empty_like(x)))
    assert np.isfinite(got).all() and got[0, 5] == 127 * 2.0 ** 121
    x = torch.full((1, 32), 65504.0, device="cuda", dtype=torch.half)
    assert (ops.Checkpoint8.empty(1, 32).store(x).load(torch.empty_like(x)) == 65504).all()


@pytest.mark.parametrize("kind", KINDS)
def test_infinities_and_nan_mark_their_block_only(ops, kind):
    x = spread(3, 200, kind, 1)
    x[:] = torch.where(torch.isfinite(x), x, 0)
    x[0, 40], x[1, 199], x[2, 64] = float("inf"), float("nan"), float("-inf")
    c = ops.Checkpoint8.empty(3, 200).store(x)
    codes, exponents = cu.encode(wide(x))
    np.testing.assert_array_equal(c.exponents.cpu().numpy(), exponents)
    np.testing.assert_array_equal(c.codes.cpu().numpy(), codes)
    got = wide(c.load(torch.empty(3, 200, device="cuda")))
    nan = np.zeros((3, 200), bool)
    nan[0, 32:64] = nan[1, 192:200] = nan[2, 64:96] = True
    np.testing.assert_array_equal(np.isnan(got), nan)


@pytest.mark.parametrize("kind", KINDS)
def test_pitched_rows(ops, kind):
    for n in (30, 1000):
        x = spread(6, n, kind, 2)
        room = torch.full((6, n + 9), 7.0, dtype=x.dtype, device="cuda")
        room[:, 5:5 + n] = x
        a, b = ops.Checkpoint8.empty(6, n).store(x), ops.Checkpoint8.empty(6, n).store(room[:, 5:5 + n])
        assert torch.equal(a.codes, b.codes) and torch.equal(a.exponents, b.exponents)
        out = torch.full((6, n + 9), 7.0, dtype=x.dtype, device="cuda")
        a.load(out[:, 5:5 + n])
        assert torch.equal(out[:, 5:5 + n], a.load(torch.empty_like(x)))
        assert (out[:, :5] == 7).all() and (out[:, 5 + n:] == 7).all()


FUNCTIONS = ["sigmoid", "relu", "leaky_relu", "linear", "tanh", "gelu"]


@pytest.mark.parametrize("func", FUNCTIONS)
@pytest.mark.parametrize("rows,n", [(1, 1), (5, 33), (64, 1000), (3, 40001)])
def test_function_backward(ops, rows, n, func):
    """The same bits as the function layer's backward pass at the kept values; from bf16 and fp16 errors rounded once."""
    r = np.random.default_rng(n)
    z = torch.from_numpy(r.normal(0, 2, (rows, n)).astype(np.float32)).cuda()
    c = ops.Checkpoint8.empty(rows, n).store(z)
    at = c.load(torch.empty_like(z))
    for kind in KINDS:
        e = torch.from_numpy(r.normal(0, 1, (rows, n))).to(getattr(torch, kind)).cuda()
        want = torch.empty(rows, n, device="cuda")
        ops.CTensorApplyFunc.Backward(want, at, e.float(), func, 0.2)
        got = torch.empty_like(e)
        ops.CTensorApplyFunc.Backward(got, c, e, func, 0.2)
        assert torch.equal(got, want.to(e.dtype))
        ops.CTensorApplyFunc.Backward(e, c, e, func, 0.2)             # in place
        assert torch.equal(got, e)
    ops.stream_status()


@pytest.mark.parametrize("func", ["sigmoid", "tanh"])
def test_function_backward_against_differences(ops, func):
    z = torch.from_numpy(np.random.default_rng(0).normal(0, 1.5, (4, 500)).astype(np.float32)).cuda()
    c = ops.Checkpoint8.empty(4, 500).store(z)
    v = cu.decode(c.codes.cpu().numpy(), c.exponents.cpu().numpy(), 500)
    f = np.tanh if func == "tanh" else lambda t: 1 / (1 + np.exp(-t))
    h = 1e-5
    got = torch.empty_like(z)
    ops.CTensorApplyFunc.Backward(got, c, torch.ones_like(z), func)
    # the derivative of either is formed from a function value that is off by a few u: 16 u absolute; the differences are off
    # by h^2/6 * 2 and by 2^-53 / h
    np.testing.assert_allclose(wide(got), (f(v + h) - f(v - h)) / (2 * h), rtol=0, atol=16 * cu.U + 1e-9)


def test_kept_signs_make_relu_exact(ops):
    z = torch.from_numpy(np.random.default_rng(1).normal(0, 1, (50, 333)).astype(np.float32)).cuda()
    z[:, ::7] *= 1e-6
    e = torch.randn_like(z)
    c = ops.Checkpoint8.empty(50, 333).store(z, keep_sign=True)
    for func in ("relu", "leaky_relu"):
        got, want = torch.empty_like(z), torch.empty_like(z)
        ops.CTensorApplyFunc.Backward(got, c, e, func)
        ops.CTensorApplyFunc.Backward(want, z, e, func)
        assert torch.equal(got, want)


@pytest.mark.parametrize("n", [200, 203])
def test_function_backward_of_gelu_is_the_stated_expression(ops, n):
    """Against (1 + tanh u + v/2 / cosh^2 u) u' / 2 in 64 bits.  In fp32 u is off by at most 4 units of 2^-24 of itself, tanhf and
    coshf by 2 ulp: tanh u by 4 |u| / cosh^2 u + 4 <= 6 units, 1 / cosh^2 u by 2 (4 |u| + 6) units of itself, which v/2 / cosh^2 u
    (at most 0.3; 0.3 |u| too) makes 6, the sums and products 4 more: less than 32 units of 1 + |u'| (u' / 2 and its own error
    of 4 units on at most 2)."""
    z = torch.from_numpy(np.random.default_rng(n).normal(0, 2, (9, n)).astype(np.float32)).cuda()
    e = torch.from_numpy(np.random.default_rng(n + 1).normal(0, 1, (9, n)).astype(np.float32)).cuda()
    c = ops.Checkpoint8.empty(9, n).store(z)
    v = cu.decode(c.codes.cpu().numpy(), c.exponents.cpu().numpy(), n)
    k, b = float(np.float32(0.7978845608)), float(np.float32(0.044715))
    u, du = k * (v + b * v ** 3), k * (1 + 3 * b * v ** 2)
    want = 0.5 * (1 + np.tanh(u) + 0.5 * v / np.cosh(u) ** 2) * du * wide(e)
    got = torch.empty_like(z)
    ops.CTensorApplyFunc.Backward(got, c, e, "gelu")
    ops.stream_status()
    cu.within(wide(got), want, 32 * cu.U * (1 + du) * np.abs(wide(e)), "gelu")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("func", FUNCTIONS)
@pytest.mark.parametrize("n", [200, 203])
def test_function_backward_of_blocks_without_values(ops, n, func, kind):
    """A block that held an infinity or a NaN is NaN in the error below: its finite values are lost, and none of them may pass for a
    negative one.  Only the linear function needs no value.  Other blocks are as ever."""
    x = torch.from_numpy(np.random.default_rng(n).normal(0, 1, (3, n)).astype(np.float32)).cuda()
    good = ops.Checkpoint8.empty(3, n).store(x, keep_sign=True)
    x[0, 40], x[1, n - 1], x[2, 64] = float("inf"), float("nan"), float("-inf")
    bad = ops.Checkpoint8.empty(3, n).store(x, keep_sign=True)
    e = torch.ones(3, n, device="cuda").to(getattr(torch, kind))
    got, want = torch.empty_like(e), torch.empty_like(e)
    ops.CTensorApplyFunc.Backward(got, bad, e, func, 0.2)
    ops.CTensorApplyFunc.Backward(want, good, e, func, 0.2)
    ops.stream_status()
    lost = torch.zeros(3, n, dtype=torch.bool, device="cuda")
    if func != "linear":
        lost[0, 32:64] = lost[1, 192:] = lost[2, 64:96] = True
    assert torch.equal(torch.isnan(got), lost)
    assert torch.equal(got[~lost], want[~lost])


WGRAD = [(1, 1, 1), (1, 40, 3), (2, 33, 64), (31, 100, 129), (64, 100, 8192), (128, 16384, 256), (200, 1000, 130), (333, 257, 65), (1000, 64, 64),
         (5000, 300, 70), (8192, 512, 384), (257, 31, 1)]


def wgrad_bound(delta, x, rows):
    """delta enters exactly (in parts of 8 bits), so do the kept values; every one of at most rows + 64 additions may truncate:
    2^-23 of the sum of magnitudes each."""
    return (rows + 64) * 2.0 ** -23 * (np.abs(delta).T @ np.abs(x))


@pytest.mark.parametrize("mode", ["TF32X3", "TF32", "FP32"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n,out", WGRAD)
def test_wgrad(ops, rows, n, out, kind, mode):
    if mode != "TF32X3" and rows * n * out > 1 << 24:
        pytest.skip("the other precision modes on the small sizes")
    ops.set_precision(getattr(ops, mode))
    try:
        r = np.random.default_rng(rows + n)
        x = torch.from_numpy(r.normal(0, 1, (rows, n)).astype(np.float32)).cuda()
        delta = torch.from_numpy(r.normal(0, 1, (rows, out)).astype(np.float32)).to(getattr(torch, kind)).cuda()
        c = ops.Checkpoint8.empty(rows, n).store(x)
        dw, db = torch.full((out, n), 5.0, device="cuda"), torch.full((out,), 5.0, device="cuda")
        ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        ops.stream_status()
        v, d = cu.decode(c.codes.cpu().numpy(), c.exponents.cpu().numpy(), n), wide(delta)
        bound, want = wgrad_bound(d, v, rows), d.T @ v
        cu.within(wide(dw), want, bound, "dweight")
        bb = (rows + 64) * 2.0 ** -23 * np.abs(d).sum(0)
        cu.within(wide(db), d.sum(0), bb, "dbias")
        first = dw.clone(), db.clone()
        ops.checkpoint_wgrad(dw, db, delta, c)                       # accumulated
        cu.within(wide(dw), 2 * want, 2 * bound + 2 * cu.U * np.abs(want), "dweight twice")
        cu.within(wide(db), 2 * d.sum(0), 2 * bb + 2 * cu.U * np.abs(d.sum(0)), "dbias twice")
        ops.checkpoint_wgrad(dw, None, delta, c, accumulate=False)   # without a bias gradient, again the same bits
        assert torch.equal(dw, first[0])
        ops.stream_status()
    finally:
        ops.set_precision(ops.TF32X3)


def test_wgrad_pitched_delta_infinities_and_nan(ops):
    rows, n, out = 100, 200, 77
    r = np.random.default_rng(5)
    c = ops.Checkpoint8.empty(rows, n).store(torch.from_numpy(r.uniform(1, 2, (rows, n)).astype(np.float32)).cuda())
    v = cu.decode(c.codes.cpu().numpy(), c.exponents.cpu().numpy(), n)
    for kind in KINDS:
        t = getattr(torch, kind)
        room = torch.full((rows, out + 9), float("nan"), dtype=t, device="cuda")
        delta = room[:, 5:5 + out]
        delta.copy_(torch.from_numpy(r.normal(0, 1, (rows, out))).to(t))
        dw, db = torch.empty(out, n, device="cuda"), torch.empty(out, device="cuda")
        ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        cu.within(wide(dw), wide(delta).T @ v, wgrad_bound(wide(delta), v, rows), kind)
        delta[17, 3], delta[20, 40], delta[99, 76] = float("inf"), float("nan"), float("-inf")
        ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        ops.stream_status()
        for got in (dw.cpu(), db.cpu().view(-1, 1)):
            assert (got[3] == float("inf")).all() and torch.isnan(got[40]).all() and (got[76] == float("-inf")).all()
            rest = [k for k in range(out) if k not in (3, 40, 76)]
            assert torch.isfinite(got[rest]).all()


def test_wgrad_largest_delta(ops):
    top = torch.finfo(torch.float32).max
    delta = torch.tensor([[top, -top, 2.0 ** -126]], device="cuda")
    c = ops.Checkpoint8.empty(1, 32).store(torch.full((1, 32), 0.5, device="cuda"))
    dw, db = torch.empty(3, 32, device="cuda"), torch.empty(3, device="cuda")
    ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
    np.testing.assert_allclose(wide(dw), np.repeat(wide(delta).T * 0.5, 32, axis=1), rtol=4 * 2.0 ** -23)
    np.testing.assert_array_equal(wide(db), wide(delta)[0])


def test_no_rows(ops):
    c = ops.Checkpoint8.empty(0, 40).store(torch.empty(0, 40, device="cuda"))
    assert c.load(torch.empty(0, 40, device="cuda")).shape == (0, 40)
    dw, db = torch.full((3, 40), 2.0, device="cuda"), torch.full((3,), 2.0, device="cuda")
    ops.checkpoint_wgrad(dw, db, torch.empty(0, 3, device="cuda"), c)
    assert (dw == 2).all() and (db == 2).all()
    ops.checkpoint_wgrad(dw, db, torch.empty(0, 3, device="cuda"), c, accumulate=False)
    ops.stream_status()
    assert (dw == 0).all() and (db == 0).all()


def test_captured_on_two_streams(ops):
    runs = []
    for k in range(2):
        delta = torch.randn(600, 200 + k, device="cuda")
        c = ops.Checkpoint8.empty(600, 500 + 40 * k).store(torch.randn(600, 500 + 40 * k, device="cuda"))
        dw, db = torch.empty(200 + k, c.n, device="cuda"), torch.empty(200 + k, device="cuda")
        ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        torch.cuda.synchronize()
        want = dw.clone(), db.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        dw.zero_(), db.zero_()
        runs.append((g, dw, db, want, delta, c, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, *_, s in runs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, dw, db, want, *_ in runs:
        assert torch.equal(dw, want[0]) and torch.equal(db, want[1])


def test_refusals(ops):
    B, x = ops.B200Error, torch.zeros(4, 64, device="cuda")
    c = ops.Checkpoint8.empty(4, 64)
    room = torch.zeros(4 * 64 + 8, dtype=torch.int8, device="cuda")
    dw, db = torch.zeros(5, 64, device="cuda"), torch.zeros(5, device="cuda")
    for bad in (lambda: c.store(x[:, :63]), lambda: c.store(x.double()), lambda: c.load(x[:3]), lambda: c.store(x.t()),
                lambda: ops.Checkpoint8(c.codes, c.exponents, 65), lambda: ops.Checkpoint8(c.codes, c.exponents.view(-1), 64),
                lambda: ops.Checkpoint8(c.codes.cpu(), c.exponents.cpu(), 64), lambda: ops.Checkpoint8(c.exponents, c.codes, 64),
                lambda: ops.Checkpoint8.empty(4, 0), lambda: ops.Checkpoint8(room[8:].view(4, 64), c.exponents, 64).store(x),
                lambda: ops.CTensorApplyFunc.Backward(x, c, x.half(), "tanh"), lambda: ops.CTensorApplyFunc.Backward(x, c, x[:, :60], "tanh"),
                lambda: ops.checkpoint_wgrad(dw, db, torch.zeros(3, 5, device="cuda"), c), lambda: ops.checkpoint_wgrad(dw[:4], db, torch.zeros(4, 5, device="cuda"), c),
                lambda: ops.checkpoint_wgrad(dw, db[:4], torch.zeros(4, 5, device="cuda"), c),
                lambda: ops.checkpoint_wgrad(dw, db, torch.zeros(4, 5, device="cuda").double(), c)):
        with pytest.raises(B):
            bad()
    ops.stream_status()


@pytest.mark.parametrize("kind,rows,n,out", [("bfloat16", 8192, 2048, 1024), ("float32", 2000, 1500, 700), ("float16", 1000, 513, 300)])
def test_wgrad_repeats_bit_for_bit(ops, kind, rows, n, out):
    """Many launches in a row: no wait of the kernel gives up, and the result is the same every time."""
    c = ops.Checkpoint8.empty(rows, n).store(torch.randn(rows, n, device="cuda"))
    delta = torch.randn(rows, out, device="cuda").to(getattr(torch, kind))
    first = None
    for i in range(60):
        dw, db = torch.empty(out, n, device="cuda"), torch.empty(out, device="cuda")
        ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        first = first or (dw, db)
        assert i % 20 or (torch.equal(dw, first[0]) and torch.equal(db, first[1]))
    ops.stream_status()


@pytest.mark.parametrize("mode", ["TF32X3", "FP32"])
@pytest.mark.parametrize("n,out", [(2, 4194304 + 131), (4194304 + 70, 2)])
def test_wgrad_of_very_many_outputs(ops, n, out, mode):
    """More than 65535 tiles of 64 in either direction, in both forms of the product.  Whole numbers: every sum is exact."""
    ops.set_precision(getattr(ops, mode))
    try:
        rows = 3
        x = torch.randint(-7, 8, (rows, n), device="cuda").float()
        delta = torch.randint(-7, 8, (rows, out), device="cuda").float()
        c = ops.Checkpoint8.empty(rows, n).store(x)
        dw, db = torch.full((out, n), 5.0, device="cuda"), torch.full((out,), 5.0, device="cuda")
        ops.checkpoint_wgrad(dw, db, delta, c)
        ops.stream_status()
        assert torch.equal(dw.double(), 5 + delta.double().t() @ x.double())
        assert torch.equal(db.double(), 5 + delta.double().sum(0))
    finally:
        ops.set_precision(ops.TF32X3)


# ---- large tensors: every loop of the kernels turns several times -----------------------------------------------------------------

def encode_there(x, keep_sign=False):
    """ckpt8_util.encode in 64 bits on the GPU (finite values)."""
    rows, n = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -n % 32)).view(rows, -1, 32)
    top = v.abs().amax(2)
    e = torch.where(top > 0, (torch.frexp(top).exponent - 1).clamp(min=-126), -126)
    b = e + 127
    b = b + ((torch.round(torch.ldexp(top, 133 - b)) > 127) & (b < 254)).int()
    q = torch.round(torch.ldexp(v, (133 - b)[:, :, None])).clamp(-127, 127)
    if keep_sign:
        q = torch.where((v < 0) & (q == 0), -1.0, q)
    return q.to(torch.int8).view(rows, -1), b.to(torch.uint8)


# more spans (32 lanes of 16 bytes, or of one value) than four for each warp of 8 x 148 blocks; one long row, rows of whole blocks,
# rows that end inside a block, rows that start anywhere
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", [(1, 6000001), (2600, 4096), (2601, 4104), (5003, 1021), (160000, 40)])
def test_large_tensors_bit_for_bit(ops, rows, n, kind):
    t = getattr(torch, kind)
    g = torch.Generator(device="cuda").manual_seed(rows)
    low, high = {"float32": (-140, 120), "bfloat16": (-125, 120), "float16": (-20, 12)}[kind]
    power = torch.randint(low, high, (rows, -(-n // 32)), device="cuda", generator=g).repeat_interleave(32, dim=1)[:, :n]
    x = torch.ldexp(torch.randn(rows, n, device="cuda", generator=g, dtype=torch.float64), power).to(t)
    for keep_sign in (False, True):
        c = ops.Checkpoint8.empty(rows, n).store(x, keep_sign=keep_sign)
        codes, exponents = encode_there(x, keep_sign)
        assert torch.equal(c.codes, codes) and torch.equal(c.exponents, exponents)
    values = torch.ldexp(codes.double(), (exponents.int() - 133).repeat_interleave(32, dim=1))[:, :n]
    at = c.load(torch.empty(rows, n, device="cuda"))
    assert torch.equal(at.double(), values)
    assert torch.equal(c.load(torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)).double(), values)
    e = torch.randn(rows, n, device="cuda", generator=g).to(t)
    for func in ("leaky_relu", "tanh"):
        want, got = torch.empty(rows, n, device="cuda"), torch.empty_like(e)
        ops.CTensorApplyFunc.Backward(want, at, e.float(), func, 0.2)
        ops.CTensorApplyFunc.Backward(got, c, e, func, 0.2)
        assert torch.equal(got, want.to(t))
    ops.stream_status()


# tiles of 256 x 256 outputs over 74 pairs of SMs, chunks of 2048 rows (bf16) or 1024, a tail of tiles split along the batch:
# 90 tiles = one round and a split tail; the same with several chunks a tile, ragged and not; 32 tiles in two units of several chunks;
# one tile in 70 units; 272 tiles = three rounds and a tail that is not split
LARGE_WGRAD = [(300, 2500, 2100), (2500, 2501, 2090), (2500, 2560, 2304), (8192, 2048, 1024), (9000, 256, 256), (5000, 4103, 4096)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n,out", LARGE_WGRAD)
def test_wgrad_of_many_tiles_and_chunks(ops, rows, n, out, kind):
    """First with whole numbers, whose sums (at most 49 rows < 2^24) are exact in any order: a tile, a chunk or a row that is left
    out or counted twice shows.  Then with any numbers: products are exact, a chunk's additions may truncate (2^-23 of the
    magnitudes each, rows of the chunk + 64 of them), and the chunks and the units of a split tile (74 at most) are added
    in fp32."""
    t = getattr(torch, kind)
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    chunk = 2048 if kind == "bfloat16" else 1024
    for whole in (True, False):
        if whole:
            x = torch.randint(-7, 8, (rows, n), device="cuda", generator=g).float()
            delta = torch.randint(-7, 8, (rows, out), device="cuda", generator=g).to(t)
        else:
            x = torch.randn(rows, n, device="cuda", generator=g)
            delta = torch.randn(rows, out, device="cuda", generator=g).to(t)
        c = ops.Checkpoint8.empty(rows, n).store(x)
        v, d = c.load(torch.empty_like(x)).double(), delta.double()
        assert not whole or torch.equal(v, x.double())
        want, want_b = d.t() @ v, d.sum(0)
        steps = (min(rows, chunk) + 64) * 2.0 ** -23 + (rows // chunk + 1 + 74) * cu.U
        bound, bound_b = (0, 0) if whole else (steps * (d.abs().t() @ v.abs()), (rows + 64) * cu.U * d.abs().sum(0))
        dw, db = torch.full((out, n), 5.0, device="cuda"), torch.full((out,), -5.0, device="cuda")
        ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        ops.stream_status()
        assert ((dw.double() - want).abs() <= bound).all() and ((db.double() - want_b).abs() <= bound_b).all()
        first = dw.clone(), db.clone()
        ops.checkpoint_wgrad(dw, db, delta, c)
        ops.stream_status()
        if whole:
            assert torch.equal(dw, 2 * first[0]) and torch.equal(db, 2 * first[1])
        else:
            assert ((dw.double() - 2 * want).abs() <= 2 * bound + 2 * cu.U * want.abs()).all()
            assert ((db.double() - 2 * want_b).abs() <= 2 * bound_b + 2 * cu.U * want_b.abs()).all()


@pytest.mark.parametrize("kind", KINDS)
def test_wgrad_empties_its_accumulator(ops, kind):
    """The tensor core truncates what does not fit 24 bits, so its sums are taken over 2048 rows (1024 in fp16 and fp32) and added to
    the output.  Sixteen rows add 63441, an odd number: 2048 rows stay below 2^23, where every sum is exact, and so are the
    multiples of 128 x 63441 that are added then.  One sum over 8192 rows would leave 2^24 behind after half of them, where
    the odd ones lose their last bit."""
    rows, n, out = 8192, 2560, 2304
    delta = torch.full((rows, out), 63.0, device="cuda")
    delta[::16] = 62.0
    c = ops.Checkpoint8.empty(rows, n).store(torch.full((rows, n), 63.0, device="cuda"))
    dw, db = torch.empty(out, n, device="cuda"), torch.empty(out, device="cuda")
    ops.checkpoint_wgrad(dw, db, delta.to(getattr(torch, kind)), c, accumulate=False)
    ops.stream_status()
    assert 63441 == 15 * 63 * 63 + 62 * 63 and 128 * 63441 < 2 ** 23
    assert (dw == 512 * 63441).all() and (db == 63 * rows - rows // 16).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n,out,launches", [(8192, 2048, 1024, 3000), (2500, 2501, 2090, 600), (200, 1000, 700, 1000)])
def test_wgrad_reads_every_stage_in_its_turn(ops, rows, n, out, launches, kind):
    """Three sets of whole numbers in turn, thousands of launches: a slot of a ring that is read before it is filled, or filled again
    before it is read, holds other rows' values or another set's, and shows."""
    sets = []
    for k in range(3):
        x = torch.randint(-7, 8, (rows, n), device="cuda").float()
        delta = torch.randint(-7, 8, (rows, out), device="cuda").to(getattr(torch, kind))
        want = (delta.double().t() @ x.double()).float()
        sets.append((delta, ops.Checkpoint8.empty(rows, n).store(x), want, delta.double().sum(0).float()))
    dw, db, wrong = torch.empty(out, n, device="cuda"), torch.empty(out, device="cuda"), torch.zeros((), dtype=torch.int64, device="cuda")
    for turn in range(launches):
        delta, c, want, want_b = sets[turn % 3]
        ops.checkpoint_wgrad(dw, db, delta, c, accumulate=False)
        wrong += (dw != want).sum() + (db != want_b).sum()
    ops.stream_status()
    assert int(wrong) == 0
