"""Layer normalisation on the GPU against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

from tests import ckpt8_util as cu

pytestmark = pytest.mark.gpu
KINDS = ["float32", "bfloat16", "float16"]
# rows x n: a single value, single rows, blocks that end early, odd lengths, the borders of the kernels' forms, long rows
SIZES = [(1, 1), (5, 2), (3, 31), (4, 32), (7, 33), (1, 256), (129, 100), (37, 1021), (300, 1024), (20, 1025), (9, 4099), (33, 8192),
         (5, 8200), (3, 16384), (4, 20001), (2, 65536), (3, 131072), (2, 300007)]


@pytest.fixture(autouse=True)
def ops():
    from cuda_cnn_gan_vae_b200 import ops
    return ops


def make(rows, n, kind, seed=0, offset=0.5):
    r = np.random.default_rng(seed + rows * 7919 + n)
    t = getattr(torch, kind)
    x = torch.from_numpy((r.normal(offset, 1.0, (rows, n)) * r.uniform(0.5, 2, (rows, 1))).astype(np.float32)).to(t).cuda()
    dy = torch.from_numpy(r.normal(0, 1, (rows, n)).astype(np.float32)).to(t).cuda()
    gamma = torch.from_numpy(r.normal(1, 0.3, n).astype(np.float32)).cuda()
    beta = torch.from_numpy(r.normal(0, 0.3, n).astype(np.float32)).cuda()
    return x, dy, gamma, beta


def host(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", SIZES)
def test_forward(ops, rows, n, kind):
    x, _, gamma, beta = make(rows, n, kind)
    got = ops.ln_forward(x, gamma, beta, 1e-5)
    ops.stream_status()
    args = (host(x), host(gamma), host(beta), float(np.float32(1e-5)))
    y, mu, r, _ = cu.ln_forward(*args)
    ey, em, er, _ = cu.ln_forward_bounds(*args, kind)
    cu.within(host(got["mean"]), mu, em, "mean")
    cu.within(host(got["rstd"]), r, er, "rstd")
    cu.within(host(got["y"]), y, ey, "y")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", SIZES)
def test_forward_checkpoint(ops, rows, n, kind):
    """The kept values are the normalised rows to half a step of their block; the outputs are those without a checkpoint."""
    x, _, gamma, beta = make(rows, n, kind, 1)
    plain = ops.ln_forward(x, gamma, beta, 1e-5)
    c = ops.Checkpoint8.empty(rows, n)
    got = ops.ln_forward(x, gamma, beta, 1e-5, checkpoint=c)
    ops.stream_status()
    assert all(torch.equal(got[k], plain[k]) for k in got)
    args = (host(x), host(gamma), host(beta), float(np.float32(1e-5)))
    xh = cu.ln_forward(*args)[3]
    exh = cu.ln_forward_bounds(*args, kind)[3]
    b = c.exponents.cpu().numpy()
    step = np.repeat(np.ldexp(1.0, b.astype(np.int64) - 133), 32, axis=1)[:, :n]
    cu.within(cu.decode(c.codes.cpu().numpy(), b, n), xh, 0.5 * step + exh, "kept")
    # the exponent is that of the block's largest value (or a neighbour's where the largest value is at a border)
    lo, hi = cu.encode(np.maximum(np.abs(xh) * (1 - 1e-3) - exh, 0))[1], cu.encode(np.abs(xh) * (1 + 1e-3) + exh)[1]
    assert (np.minimum(lo, hi) <= b).all() and (b <= hi).all()
    assert not c.codes.cpu().numpy().reshape(rows, -1)[:, n:].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows,n", SIZES)
def test_backward(ops, rows, n, kind, accumulate):
    x, dy, gamma, beta = make(rows, n, kind, 2)
    mu = x.double().mean(1).float()
    rstd = (1 / (x.double().var(1, correction=0) + 1e-5).sqrt()).float()
    dgamma, dbeta = (torch.full((n,), 3.0, device="cuda") for _ in range(2))
    dx = ops.ln_backward(dy, x, mu, rstd, gamma, dgamma, dbeta, accumulate=accumulate)
    ops.stream_status()
    xh = (host(x) - host(mu)[:, None]) * host(rstd)[:, None]
    want = cu.ln_backward(host(dy), xh, host(rstd), host(gamma))
    edx, edg, edb = cu.ln_backward_bounds(host(dy), xh, host(rstd), host(gamma), kind)
    base = 3.0 if accumulate else 0.0
    cu.within(host(dx), want[0], edx, "dx")
    cu.within(host(dgamma), want[1] + base, edg + cu.U * np.abs(want[1] + base), "dgamma")
    cu.within(host(dbeta), want[2] + base, edb + cu.U * np.abs(want[2] + base), "dbeta")
    # without the parameters' gradients: the same dx, nothing else written
    keep = dgamma.clone(), dbeta.clone()
    again = ops.ln_backward(dy, x, mu, rstd, gamma, dgamma, dbeta, create_delta_weight=False)
    assert torch.equal(again, dx) and torch.equal(dgamma, keep[0]) and torch.equal(dbeta, keep[1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", SIZES)
def test_backward_from_checkpoint(ops, rows, n, kind):
    x, dy, gamma, beta = make(rows, n, kind, 3)
    c = ops.Checkpoint8.empty(rows, n)
    got = ops.ln_forward(x, gamma, beta, 1e-5, checkpoint=c)
    dgamma, dbeta = (torch.zeros(n, device="cuda") for _ in range(2))
    dx = ops.ln_backward(dy, c, None, got["rstd"], gamma, dgamma, dbeta)
    ops.stream_status()
    xh = cu.decode(c.codes.cpu().numpy(), c.exponents.cpu().numpy(), n)
    want = cu.ln_backward(host(dy), xh, host(got["rstd"]), host(gamma))
    edx, edg, edb = cu.ln_backward_bounds(host(dy), xh, host(got["rstd"]), host(gamma), kind)
    cu.within(host(dx), want[0], edx, "dx")
    cu.within(host(dgamma), want[1], edg + cu.U * np.abs(want[1]), "dgamma")
    cu.within(host(dbeta), want[2], edb + cu.U * np.abs(want[2]), "dbeta")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 9, 33, 517, 1021, 4099])
def test_backward_at_the_ends_of_a_tensor(ops, n, kind, checkpoint):
    """Rows whose first and last 16 bytes they share with other rows, or with what lies around the tensor: it is NaN and must
    neither count nor change."""
    t = getattr(torch, kind)

    def around(x, start):
        wide = torch.full((x.numel() + 32,), float("nan"), dtype=t, device="cuda")
        inner = wide[start:start + x.numel()].view(x.shape)
        inner.copy_(x)
        return wide, inner

    for rows in (1, 2, 9, 40):
        x, dy, gamma, _ = make(rows, n, kind, 7)
        mean, var = x.double().mean(1), x.double().var(1, correction=0)
        rstd = (1 / (var + 1e-5).sqrt()).float()
        mean = mean.float()
        xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
        c = None
        if checkpoint:
            c = ops.Checkpoint8.empty(rows, n).store(xh.float())
            xh = c.load(torch.empty(rows, n, device="cuda")).double()
        for start in (0, 1, 5, 8, 15):
            wide_dy, in_dy = around(dy, start)
            _, in_x = around(x, (3 * start + 1) % 16)
            wide_dx, dx = around(torch.zeros_like(dy), start)
            dg, db = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
            ops.ln_backward(in_dy, c if checkpoint else in_x, None if checkpoint else mean, rstd, gamma, dg, db, dx=dx)
            ops.stream_status()
            want, g, b = cu.ln_backward(host(dy), host(xh), host(rstd), host(gamma))
            e, eg, eb = cu.ln_backward_bounds(host(dy), host(xh), host(rstd), host(gamma), kind)
            cu.within(host(dx), want, e, "dx")
            cu.within(host(dg), g, eg + cu.U * np.abs(g), "dgamma")
            cu.within(host(db), b, eb + cu.U * np.abs(b), "dbeta")
            outside = torch.isnan(wide_dx)
            assert outside[:start].all() and outside[start + dx.numel():].all() and int(outside.sum()) == 32


@pytest.mark.parametrize("n", [24, 1000, 8192, 40000])
def test_pitched_rows_and_untouched_surroundings(ops, n):
    """Rows inside wider matrices, starting at odd elements: nothing outside the rows is read into the result or written."""
    rows = 6
    for kind in KINDS:
        t = getattr(torch, kind)
        x, dy, gamma, beta = make(rows, n, kind, 4)
        wide = [torch.full((rows, n + 7 + k), float("nan"), dtype=t, device="cuda") for k in range(4)]
        vx, vdy, vy, vdx = (w[:, 3:3 + n] for w in wide)
        vx.copy_(x), vdy.copy_(dy)
        want = ops.ln_forward(x, gamma, beta, 1e-5)
        got = ops.ln_forward(vx, gamma, beta, 1e-5, y=vy)
        cu.within(host(got["y"]), host(want["y"]), cu.ln_forward_bounds(host(x), host(gamma), host(beta), 1e-5, kind)[0] * 2, "y")
        dg, db, dg2, db2 = (torch.zeros(n, device="cuda") for _ in range(4))
        ops.ln_backward(dy, x, want["mean"], want["rstd"], gamma, dg, db)
        ops.ln_backward(vdy, vx, want["mean"], want["rstd"], gamma, dg2, db2, dx=vdx)
        ops.stream_status()
        xh = (host(x) - host(want["mean"])[:, None]) * host(want["rstd"])[:, None]
        bounds = cu.ln_backward_bounds(host(dy), xh, host(want["rstd"]), host(gamma), kind)
        cu.within(host(vdx), cu.ln_backward(host(dy), xh, host(want["rstd"]), host(gamma))[0], bounds[0], "dx")
        cu.within(host(dg2), host(dg), 2 * bounds[1], "dgamma")
        cu.within(host(db2), host(db), 2 * bounds[2], "dbeta")
        for w in wide[2:]:
            assert torch.isnan(w[:, :3]).all() and torch.isnan(w[:, 3 + n:]).all()


@pytest.mark.parametrize("n", [100, 1024, 8192, 20000, 300000])
def test_in_place(ops, n):
    x, dy, gamma, beta = make(5, n, "float32", 5)
    want = ops.ln_forward(x, gamma, beta, 1e-5)
    dg, db, dg2, db2 = (torch.zeros(n, device="cuda") for _ in range(4))
    dx = ops.ln_backward(dy, x, want["mean"], want["rstd"], gamma, dg, db)
    for target in ("dy", "x"):
        a, b = dy.clone(), x.clone()
        dg2.zero_(), db2.zero_()
        out = a if target == "dy" else b
        ops.ln_backward(a, b, want["mean"], want["rstd"], gamma, dg2, db2, dx=out)
        assert torch.equal(out, dx) and torch.equal(dg, dg2) and torch.equal(db, db2)
    y = x.clone()
    assert torch.equal(ops.ln_forward(y, gamma, beta, 1e-5, y=y)["y"], want["y"])
    ops.stream_status()


def test_constant_rows_infinities_and_nan(ops):
    """A constant row has no deviation (y = beta); a row with an infinity or a NaN gives NaN, its neighbours are untouched."""
    for n in (40, 1000, 9000):
        x, dy, gamma, beta = make(6, n, "float32", 6)
        x[1] = 4.0
        x[3, n // 2] = float("inf")
        x[4, n - 1] = float("nan")
        c = ops.Checkpoint8.empty(6, n)
        got = ops.ln_forward(x, gamma, beta, 1e-5, checkpoint=c)
        ops.stream_status()
        assert torch.equal(got["y"][1], beta)
        assert torch.isnan(got["y"][3]).all() and torch.isnan(got["y"][4]).all()
        for k in (0, 2, 5):
            alone = ops.ln_forward(x[k:k + 1], gamma, beta, 1e-5)
            assert torch.equal(alone["y"][0], got["y"][k])
        kept = c.load(torch.empty(6, n, device="cuda"))
        assert torch.isnan(kept[3]).all() and torch.isnan(kept[4]).all() and (kept[1] == 0).all()
        assert torch.isfinite(kept[[0, 2, 5]]).all()


def test_large_mean(ops):
    """The variance comes from deviations about the mean: a mean of 1000 deviations costs no more than its own rounding."""
    x, _, gamma, beta = make(8, 5000, "float32", 7, offset=0.0)
    x += 1000.0
    args = (host(x), host(gamma), host(beta), 1e-5)
    got = ops.ln_forward(x, gamma, beta, 1e-5)
    cu.within(host(got["y"]), cu.ln_forward(*args)[0], cu.ln_forward_bounds(*args, "float32")[0], "y")
    cu.within(host(got["rstd"]), cu.ln_forward(*args)[2], cu.ln_forward_bounds(*args, "float32")[2], "rstd")


@pytest.mark.parametrize("n", [48, 3000])
def test_gradient_against_differences(ops, n):
    """Directional derivative of sum(w * y) by central differences of the 64-bit forward formula."""
    rows, h = 4, 1e-4
    x, w, gamma, beta = make(rows, n, "float32", 8)
    got = ops.ln_forward(x, gamma, beta, 1e-5)
    dg, db = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    dx = ops.ln_backward(w, x, got["mean"], got["rstd"], gamma, dg, db)
    r = np.random.default_rng(3)
    f = lambda X, G, B: float((cu.ln_forward(X, G, B, 1e-5)[0] * host(w)).sum())  # noqa: E731
    X, G, B = host(x), host(gamma), host(beta)
    for grad, move in ((host(dx), 0), (host(dg), 1), (host(db), 2)):
        d = r.normal(0, 1, grad.shape)
        args = [[X, G, B], [X, G, B]]
        args[0][move] = args[0][move] + h * d
        args[1][move] = args[1][move] - h * d
        want = (f(*args[0]) - f(*args[1])) / (2 * h)
        # the differences are off by h^2/6 times a third derivative (of order |w||d|^3 r^3 per value: below 1e-6 of the sum
        # of magnitudes), the gradient by rounding (about (n/32 + 20) u of the same sum)
        assert abs(want - (grad * d).sum()) <= (1e-6 + (n / 32 + 20) * cu.U) * 10 * np.abs(grad * d).sum() + 1e-6, move


def test_runs_repeat_bit_for_bit(ops):
    for rows, n in ((4000, 700), (50, 30000)):
        x, dy, gamma, beta = make(rows, n, "bfloat16", 9)
        got = ops.ln_forward(x, gamma, beta)
        outs = []
        for _ in range(3):
            dg, db = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
            outs.append((ops.ln_backward(dy, x, got["mean"], got["rstd"], gamma, dg, db), dg, db))
        for o in outs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_no_rows(ops):
    gamma = torch.ones(33, device="cuda")
    empty = torch.empty(0, 33, device="cuda")
    got = ops.ln_forward(empty, gamma, gamma)
    assert got["y"].shape == (0, 33)
    dg, db = torch.full((33,), 2.0, device="cuda"), torch.full((33,), 2.0, device="cuda")
    ops.ln_backward(empty, empty, got["mean"], got["rstd"], gamma, dg, db)
    assert (dg == 2).all() and (db == 2).all()
    ops.ln_backward(empty, empty, got["mean"], got["rstd"], gamma, dg, db, accumulate=False)
    ops.stream_status()
    assert (dg == 0).all() and (db == 0).all()


def test_captured_and_replayed_on_two_streams(ops):
    """Two captured passes with workspaces of their own, replayed at the same time on two streams."""
    graphs, results, wants = [], [], []
    for k in range(2):
        x, dy, gamma, beta = make(700, 900 + 64 * k, "float32", 10 + k)
        n = x.shape[1]
        dg, db = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        mean, rstd, y, dx = torch.empty(700, device="cuda"), torch.empty(700, device="cuda"), torch.empty_like(x), torch.empty_like(x)

        def step():
            ops.ln_forward(x, gamma, beta, y=y, mean=mean, rstd=rstd)
            ops.ln_backward(dy, x, mean, rstd, gamma, dg, db, accumulate=False, dx=dx)
        step()
        torch.cuda.synchronize()
        wants.append([t.clone() for t in (y, dx, dg, db)])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
        results.append((y, dx, dg, db, x, dy, gamma, beta, mean, rstd))
        for t in (y, dx, dg, db):
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for r, w in zip(results, wants):
        assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_refusals(ops):
    x, dy, gamma, beta = make(4, 64, "float32", 11)
    B = ops.B200Error
    for bad in (lambda: ops.ln_forward(x.double(), gamma, beta),
                lambda: ops.ln_forward(x.cpu(), gamma, beta),
                lambda: ops.ln_forward(x.t(), gamma, beta),
                lambda: ops.ln_forward(x, gamma[:-1], beta),
                lambda: ops.ln_forward(x, gamma.half(), beta),
                lambda: ops.ln_forward(x, gamma, beta, eps=0.0),
                lambda: ops.ln_forward(x, gamma, beta, eps=float("nan")),
                lambda: ops.ln_forward(x, gamma, beta, y=torch.empty(4, 65, device="cuda")),
                lambda: ops.ln_forward(x, gamma, beta, y=torch.empty(4, 64, device="cuda", dtype=torch.half)),
                lambda: ops.ln_forward(x, gamma, beta, checkpoint=ops.Checkpoint8.empty(4, 63)),
                lambda: ops.ln_forward(x.expand(4, 64)[:1].expand(4, 64), gamma, beta),
                lambda: ops.ln_backward(dy, x, gamma[:3], gamma[:4], gamma, gamma.clone(), beta.clone()),
                lambda: ops.ln_backward(dy, x, gamma[:4], gamma[:4], gamma, gamma.clone(), None),
                lambda: ops.ln_backward(dy, x, gamma[:4], gamma[:4], gamma, gamma.clone(), beta.clone(), workspace=torch.empty(16, device="cuda")),
                lambda: ops.ln_backward(dy, ops.Checkpoint8.empty(3, 64), None, gamma[:4], gamma, gamma.clone(), beta.clone())):
        with pytest.raises(B):
            bad()
    ops.stream_status()


@pytest.mark.parametrize("n", [1000, 20000])
def test_an_infinity_in_a_row_is_its_mean(ops, n):
    x, _, gamma, beta = make(5, n, "float32", 12)
    x[1, n // 3], x[2, n - 2], x[3, 7], x[3, 9] = float("inf"), float("-inf"), float("inf"), float("-inf")
    got = ops.ln_forward(x, gamma, beta)
    mean = got["mean"].cpu()
    assert mean[1] == float("inf") and mean[2] == float("-inf") and torch.isnan(mean[3]) and torch.isfinite(mean[[0, 4]]).all()
    assert torch.isnan(got["y"][1:4]).all() and torch.isfinite(got["y"][[0, 4]]).all()


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [9000, 20000, 131072])
def test_large_magnitudes(ops, n, kind):
    """Means whose square leaves fp32 and deviations whose square does not.  Constant rows of 2^66: every sum of up to 32 of them is exact,
    so is every mean, and the deviation is 0.  Alternating rows m (1 +- 2^-7), both exact in bf16: m^2 times a count of values is beyond
    fp32 (2^120 at least, times thousands), the sum of squared deviations is not (2^108 times 2^17 at most); compared with the
    formula, to the bounds of the other sizes."""
    t = getattr(torch, kind)
    gamma, beta = make(1, n, kind, 13)[2:]
    x = torch.full((2, n), 2.0 ** 66, dtype=t, device="cuda")
    x[1] = -x[1]
    got = ops.ln_forward(x, gamma, beta, 1e-5)
    ops.stream_status()
    assert torch.equal(got["mean"], x[:, 0].float())
    assert torch.equal(got["y"], beta.to(t).expand(2, n))
    np.testing.assert_allclose(host(got["rstd"]), float(np.float32(1e-5)) ** -0.5, rtol=3 * cu.U)
    sign = torch.where(torch.arange(n, device="cuda") % 2 == 0, 1.0, -1.0)
    x = torch.stack([2.0 ** 61 * (1 + sign * 2.0 ** -7), -(2.0 ** 60) * (1 + sign * 2.0 ** -7)]).to(t)
    args = (host(x), host(gamma), host(beta), float(np.float32(1e-5)))
    got = ops.ln_forward(x, gamma, beta, 1e-5)
    ops.stream_status()
    y, mu, r, _ = cu.ln_forward(*args)
    ey, em, er, _ = cu.ln_forward_bounds(*args, kind)
    cu.within(host(got["mean"]), mu, em, "mean")
    cu.within(host(got["rstd"]), r, er, "rstd")
    cu.within(host(got["y"]), y, ey, "y")


# ---- many rows: every loop down the rows turns several times -------------------------------------------------------------------

def close(got, want, bound, name):
    off = (got.double() - want).abs() - bound
    assert not torch.isnan(off).any(), name
    worst = int(off.argmax())
    assert off.max() <= 0, f"{name}[{worst}]: {got.flatten()[worst]} against {want.flatten()[worst]}, over the bound by {off.max()}"


# Rows for a team of the one-pass backward (148 SMs; a team of 32 threads up to 512 values, 64 up to 1024, ... 512 up to 8192, 512
# threads a block): 13, 11, 16, 17, 17, 28, where its ring has 3 to 8 slots; then rows of two passes in several groups, with both joins
MANY = [(30000, 100), (12000, 1021), (9000, 2048), (5000, 4099), (2500, 8192), (66000, 33), (150, 9001), (150, 16384), (61, 20001), (40, 65536)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("rows,n", MANY)
def test_backward_of_many_rows(ops, rows, n, kind, checkpoint):
    """Errors and normalised values are whole numbers, means and inverse deviations such that both are exact in every type: each
    product and each sum over the rows (at most 9 rows < 2^24) is exact, so a row that is left out or counted twice shows in
    dgamma or dbeta.  dx by the bounds of the other sizes."""
    t = getattr(torch, kind)
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    xh = torch.randint(-3, 4, (rows, n), device="cuda", generator=g).float()
    dy = torch.randint(-3, 4, (rows, n), device="cuda", generator=g).to(t)
    mean = torch.randint(-2, 3, (rows,), device="cuda", generator=g).float()
    rstd = torch.exp2(torch.randint(-1, 2, (rows,), device="cuda", generator=g).float())
    gamma = 1 + 0.3 * torch.randn(n, device="cuda", generator=g)
    x = (xh / rstd[:, None] + mean[:, None]).to(t)
    source = ops.Checkpoint8.empty(rows, n).store(xh) if checkpoint else x
    dgamma, dbeta = torch.full((n,), 7.0, device="cuda"), torch.full((n,), -7.0, device="cuda")
    dx = ops.ln_backward(dy, source, mean, rstd, gamma, dgamma, dbeta)
    ops.stream_status()
    xh, r = xh.double(), rstd.double()[:, None]
    assert torch.equal(dgamma.double(), 7 + (dy.double() * xh).sum(0))
    assert torch.equal(dbeta.double(), dy.double().sum(0) - 7)
    gg = dy.double() * gamma.double()
    c1, c2 = gg.mean(1, keepdim=True), (gg * xh).mean(1, keepdim=True)
    want = r * (gg - c1 - xh * c2)
    # as in ckpt8_util.ln_backward_bounds
    k, a1, a2 = cu.sum_steps(n), gg.abs().mean(1, keepdim=True), (gg * xh).abs().mean(1, keepdim=True)
    e = r * ((k + 5) * cu.U * (a1 + xh.abs() * a2) + 5 * cu.U * (gg.abs() + a1 + xh.abs() * a2)) + 2 * cu.U * want.abs()
    close(dx, want, e + cu.HALF_STEP[kind] * (want.abs() + e) + cu.TINY[kind], "dx")
    # written in place of what was there, and again, with the same bits
    other = ops.ln_backward(dy, source, mean, rstd, gamma, dgamma, dbeta, accumulate=False)
    assert torch.equal(other, dx)
    assert torch.equal(dgamma.double(), (dy.double() * xh).sum(0)) and torch.equal(dbeta.double(), dy.double().sum(0))


# more rows than the grid has teams (24 blocks for each of 148 SMs, of four rows up to 512 values, else of one), then long rows in
# several groups
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", [(33000, 100), (9000, 1000), (9000, 1021), (3700, 4099), (3600, 9001), (3600, 16384), (150, 20001), (70, 65536), (90, 20000)])
def test_forward_of_many_rows(ops, rows, n, kind):
    t = getattr(torch, kind)
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x = ((torch.randn(rows, n, device="cuda", generator=g) + 0.5) * (0.5 + torch.rand(rows, 1, device="cuda", generator=g))).to(t)
    gamma, beta = 1 + 0.3 * torch.randn(n, device="cuda", generator=g), 0.3 * torch.randn(n, device="cuda", generator=g)
    c = ops.Checkpoint8.empty(rows, n)
    got = ops.ln_forward(x, gamma, beta, 1e-5, checkpoint=c)
    ops.stream_status()
    plain = ops.ln_forward(x, gamma, beta, 1e-5)
    assert all(torch.equal(got[name], plain[name]) for name in got)
    xd = x.double()
    var, mu = torch.var_mean(xd, 1, correction=0)
    r = 1 / (var + float(np.float32(1e-5))).sqrt()
    # as in ckpt8_util.ln_forward_bounds
    k = cu.sum_steps(n)
    m = (k + 2) * cu.U * xd.abs().mean(1)
    rel = 0.5 * ((k + 4) * cu.U + (m * r) ** 2) + 3 * cu.U
    close(got["mean"], mu, m + cu.U * mu.abs(), "mean")
    close(got["rstd"], r, r * rel, "rstd")
    xh = (xd - mu[:, None]) * r[:, None]
    del xd
    e = xh.abs() * (rel + 3 * cu.U)[:, None] + (m * r)[:, None] * 1.01
    kept = c.load(torch.empty(rows, n, device="cuda"))
    step = torch.exp2(c.exponents.double() - 133).repeat_interleave(32, dim=1)[:, :n]
    close(kept, xh, 0.5 * step + e, "kept")
    del step, kept
    y = xh * gamma.double() + beta.double()
    e = gamma.double().abs() * e + 2 * cu.U * ((gamma.double() * xh).abs() + y.abs())
    close(got["y"], y, e + cu.HALF_STEP[kind] * (y.abs() + e) + cu.TINY[kind], "y")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("rows,n", [(9000, 100), (9000, 1021), (6000, 2048), (2500, 8192)])
def test_backward_reads_every_row_in_its_turn(ops, rows, n, kind, checkpoint):
    """Three sets of whole numbers in turn, hundreds of launches: a slot of a team's ring that is read before it is filled, or filled again
    before it is read, holds another row's values, and shows."""
    t, sets = getattr(torch, kind), []
    for k in range(3):
        g = torch.Generator(device="cuda").manual_seed(k)
        xh = torch.randint(-3, 4, (rows, n), device="cuda", generator=g).float()
        dy = torch.randint(-3, 4, (rows, n), device="cuda", generator=g).to(t)
        gamma = torch.randint(1, 4, (n,), device="cuda", generator=g).float()
        sets.append((dy, ops.Checkpoint8.empty(rows, n).store(xh) if checkpoint else xh.to(t), gamma, (dy.double() * xh.double()).sum(0).float(),
                     dy.double().sum(0).float()))
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    dg, db, dx = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty(rows, n, device="cuda", dtype=t)
    first = [ops.ln_backward(s[0], s[1], mean, rstd, s[2], dg, db, accumulate=False) for s in sets]
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for turn in range(300):
        dy, source, gamma, want_g, want_b = sets[turn % 3]
        ops.ln_backward(dy, source, mean, rstd, gamma, dg, db, accumulate=False, dx=dx)
        wrong += (dg != want_g).sum() + (db != want_b).sum() + (dx != first[turn % 3]).sum()
    ops.stream_status()
    assert int(wrong) == 0
