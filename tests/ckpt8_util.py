"""The 8-bit checkpoint format and layer normalisation restated in numpy with 64-bit arithmetic, and the error bounds that the
GPU tests use."""
import numpy as np

U = 2.0 ** -24                       # half a step of fp32, relative
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}    # the smallest step of the type


def encode(x, keep_sign=False):
    """codes [rows, 32 * blocks] int8 and exponents [rows, blocks] uint8 of x (any float type), from the definition."""
    x = np.asarray(x, np.float64)
    rows, n = x.shape
    blocks = -(-n // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :n] = x
    v = v.reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(2)
    v = np.where(bad[:, :, None], 0.0, v)
    top = np.abs(v).max(2)
    e = np.where(top > 0, np.maximum(np.frexp(top)[1] - 1, -126), -126)      # 2^e <= top < 2^(e+1)
    b = e + 127
    grow = (np.rint(np.ldexp(top, 133 - b)) > 127) & (b < 254)
    b = b + grow
    q = np.rint(np.ldexp(v, (133 - b)[:, :, None]))
    q = np.clip(q, -127, 127)
    if keep_sign:
        q = np.where((v < 0) & (q == 0), -1, q)
    b = np.where(bad, 255, b)
    return q.astype(np.int8).reshape(rows, -1), b.astype(np.uint8)


def decode(codes, exponents, n):
    rows, blocks = exponents.shape
    b = exponents.astype(np.int64)
    v = np.ldexp(codes.reshape(rows, blocks, 32).astype(np.float64), (b - 133)[:, :, None])
    v[b == 255] = np.nan
    return v.reshape(rows, -1)[:, :n]


def sum_steps(n):
    """Additions on the longest path of a row sum: no form of the kernels gives one thread more than n/32 values in sequence
    (a warp holds a row at least), and 16 more join the threads (5 in a warp, 5 across warps, the rest across blocks)."""
    return n / 32 + 16


def ln_forward(x, gamma, beta, eps):
    x = np.asarray(x, np.float64)
    mu = x.mean(1, keepdims=True)
    var = ((x - mu) ** 2).mean(1, keepdims=True)
    r = 1 / np.sqrt(var + eps)
    xh = (x - mu) * r
    return xh * gamma + beta, mu[:, 0], r[:, 0], xh


def ln_forward_bounds(x, gamma, beta, eps, kind):
    """Largest possible errors of y, mean, rstd and xhat: the sum of n terms is off by at most k u sum|x|; the sum of squares
    about a mean that is off by m is the true one plus n m^2, itself off by (k + 3) u; a square root and a division add 2 u."""
    x = np.asarray(x, np.float64)
    y, mu, r, xh = ln_forward(x, gamma, beta, eps)
    k = sum_steps(x.shape[1])
    m = (k + 2) * U * np.abs(x).mean(1)
    rel = 0.5 * ((k + 4) * U + (m * r) ** 2) + 3 * U
    e_xh = np.abs(xh) * (rel + 3 * U)[:, None] + (m * r)[:, None] * 1.01
    e_y = np.abs(gamma) * e_xh + 2 * U * (np.abs(gamma * xh) + np.abs(y))
    return e_y + HALF_STEP[kind] * (np.abs(y) + e_y) + TINY[kind], m + U * np.abs(mu), r * rel, e_xh


def ln_backward(dy, xh, rstd, gamma):
    dy, xh, r = np.asarray(dy, np.float64), np.asarray(xh, np.float64), np.asarray(rstd, np.float64)[:, None]
    g = dy * gamma
    c1, c2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    return r * (g - c1 - xh * c2), (dy * xh).sum(0), dy.sum(0)


def ln_backward_bounds(dy, xh, rstd, gamma, kind):
    """xhat is off by 2 u of itself (one subtraction of given numbers, one product), a row's sums by (k + 5) u of the sum of
    magnitudes, a column sum of m terms in any order by (m + 4) u of its sum of magnitudes."""
    dy, xh, r = np.asarray(dy, np.float64), np.asarray(xh, np.float64), np.abs(np.asarray(rstd, np.float64))[:, None]
    g = dy * gamma
    k = sum_steps(dy.shape[1])
    a1, a2 = np.abs(g).mean(1, keepdims=True), np.abs(g * xh).mean(1, keepdims=True)
    e = (k + 5) * U * (a1 + np.abs(xh) * a2) + 5 * U * (np.abs(g) + a1 + np.abs(xh) * a2)
    dx, dg, db = ln_backward(dy, xh, rstd, gamma)
    e_dx = r * e + 2 * U * np.abs(dx)
    m = dy.shape[0]
    return e_dx + HALF_STEP[kind] * (np.abs(dx) + e_dx) + TINY[kind], (m + 4) * U * np.abs(dy * xh).sum(0), (m + 4) * U * np.abs(dy).sum(0)


def within(got, want, bound, name):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    off = np.abs(got - want) - bound
    assert got.shape == want.shape and not np.isnan(got).any(), name
    worst = np.unravel_index(np.argmax(off), off.shape)
    assert off[worst] <= 0, f"{name}{worst}: {got[worst]!r} against {want[worst]!r}, bound {np.broadcast_to(bound, off.shape)[worst]!r}"
