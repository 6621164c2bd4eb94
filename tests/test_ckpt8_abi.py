"""The layer-normalisation and checkpoint entry points refuse bad arguments before they touch the GPU."""
import ctypes as C

import numpy as np
import pytest

from tests import ckpt8_util as cu

P = C.c_void_p(1 << 20)              # never dereferenced: every call here is refused on the host
ODD = C.c_void_p((1 << 20) + 2)
ARG, SHAPE, NOMEM = 2, 1, 5


@pytest.fixture(scope="module")
def lib():
    from cuda_cnn_gan_vae_b200 import build, lib as L
    build.build()
    return L.load()


def test_ln_forward_refusals(lib):
    def call(y=P, codes=None, exps=None, x=P, gamma=P, beta=P, kind=0, rows=4, n=64, xp=64, yp=64, eps=1e-5):
        return lib.b200_ln_forward(y, P, P, codes, exps, x, gamma, beta, kind, rows, n, xp, yp, eps, None)
    assert call(kind=3) == ARG and call(kind=-1) == ARG
    assert call(eps=0.0) == ARG and call(eps=float("nan")) == ARG and call(eps=-1.0) == ARG
    assert call(rows=-1) == SHAPE and call(n=0) == SHAPE and call(n=1 << 31) == SHAPE
    assert call(x=None) == ARG and call(y=None) == ARG and call(gamma=None) == ARG and call(beta=None) == ARG
    assert call(codes=P) == ARG and call(exps=P) == ARG and call(codes=ODD, exps=P) == ARG
    assert call(xp=63) == SHAPE and call(yp=63) == SHAPE and call(x=ODD) == ARG
    assert b"aligned" in lib.b200_last_error()
    assert call(rows=0, x=None, y=None, gamma=None) == 0


def test_ln_backward_refusals(lib):
    need = lib.b200_ln_backward_workspace(4, 64)
    assert need >= 8 * 64 and lib.b200_ln_backward_workspace(0, 64) == 0

    def call(dx=P, dg=P, db=P, dy=P, x=P, mean=P, rstd=P, codes=None, exps=None, gamma=P, kind=0, rows=4, n=64, pitch=64, create=1, ws=P, size=need):
        return lib.b200_ln_backward(dx, dg, db, dy, x, mean, rstd, codes, exps, gamma, kind, rows, n, pitch, 64, 64, create, 0, ws, size, None)
    assert call(kind=7) == ARG and call(rows=-2) == SHAPE and call(n=0) == SHAPE
    assert call(dg=None) == ARG and call(db=None) == ARG and call(rstd=None) == ARG and call(gamma=None) == ARG and call(mean=None) == ARG
    assert call(codes=P, exps=P) == ARG and call(x=None) == ARG           # both sources, none
    assert call(x=None, codes=P) == ARG and call(dx=None) == ARG and call(dy=None) == ARG and call(pitch=10) == SHAPE
    assert call(ws=None) == ARG and call(ws=ODD) == ARG and call(size=need - 1) == NOMEM
    assert call(rows=0, create=0, dx=None, x=None) == 0


def test_ckpt8_refusals(lib):
    assert lib.b200_ckpt8_store(P, P, P, 9, 4, 64, 64, 0, None) == ARG
    assert lib.b200_ckpt8_store(P, P, P, 0, -4, 64, 64, 0, None) == SHAPE
    assert lib.b200_ckpt8_store(ODD, P, P, 0, 4, 64, 64, 0, None) == ARG
    assert lib.b200_ckpt8_store(P, None, P, 0, 4, 64, 64, 0, None) == ARG
    assert lib.b200_ckpt8_store(P, P, P, 0, 4, 64, 60, 0, None) == SHAPE
    assert lib.b200_ckpt8_load(None, P, P, 0, 4, 64, 64, None) == ARG
    assert lib.b200_ckpt8_load(P, P, P, 1, 4, 0, 64, None) == SHAPE
    assert lib.b200_ckpt8_activation_backward(P, P, P, P, 0, 4, 64, 64, 64, 6, 0.1, None) == ARG
    assert lib.b200_ckpt8_activation_backward(P, P, P, None, 0, 4, 64, 64, 64, 1, 0.1, None) == ARG
    assert lib.b200_ckpt8_activation_backward(P, P, P, P, 0, 4, 64, 64, 63, 1, 0.1, None) == SHAPE


def test_wgrad_refusals(lib):
    def call(dw=P, delta=P, codes=P, kind=0, rows=4, out=8, n=64, pitch=8, ws=P, size=1 << 40):
        return lib.b200_ckpt8_wgrad(dw, None, 0, delta, codes, P, kind, rows, out, n, pitch, ws, size, None)
    assert call(kind=4) == ARG and call(rows=-1) == SHAPE and call(out=0) == SHAPE and call(n=0) == SHAPE
    assert call(dw=None) == ARG and call(delta=None) == ARG and call(codes=None) == ARG and call(codes=ODD) == ARG and call(pitch=7) == SHAPE


def test_the_restated_format_keeps_its_promises():
    """Half a step at most, 1/127 of the block's largest magnitude; signs kept on demand; 8 bits exact in bf16."""
    r = np.random.default_rng(0)
    x = (r.normal(0, 1, (40, 333)) * np.ldexp(1.0, r.integers(-120, 120, (40, 1)))).astype(np.float32)
    codes, exponents = cu.encode(x)
    v = cu.decode(codes, exponents, 333)
    top = np.repeat(np.abs(np.pad(x, ((0, 0), (0, 19))).reshape(40, -1, 32)).max(2), 32, axis=1)[:, :333]
    assert (np.abs(v - x) <= top / 127).all()
    assert (np.abs(codes) <= 127).all() and (np.abs(codes.reshape(40, -1, 32)).max(2) >= 64).all()
    kept = cu.decode(*cu.encode(x, keep_sign=True), 333)
    assert ((kept < 0) == (x < 0)).all()
    torch = pytest.importorskip("torch")
    assert np.array_equal(torch.from_numpy(v).bfloat16().double().numpy(), v)


@pytest.mark.parametrize("shape", [(2 ** 32 + 5, 1), (2 ** 32 + 4, 1, 1), (2 ** 31 - 65535, 2), (3, 2 ** 32 + 64), (3, 2 ** 16, 2 ** 16 + 1)])
def test_sizes_beyond_the_interface_are_refused_and_not_cut_to_32_bits(monkeypatch, shape):
    """Tensors without memory (nothing may look at their data): more rows, or longer ones, than the library takes."""
    torch = pytest.importorskip("torch")
    from torch._subclasses.fake_tensor import FakeTensorMode
    from cuda_cnn_gan_vae_b200 import ops
    monkeypatch.setattr(ops, "_device", lambda: 0)
    with FakeTensorMode():
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        n = x[0].numel()
        blocks = -(-n // 32)
        gamma = torch.empty(n, device="cuda")
        kept = ops.Checkpoint8(torch.empty(shape[0], 32 * blocks, dtype=torch.int8, device="cuda"),
                               torch.empty(shape[0], blocks, dtype=torch.uint8, device="cuda"), n)
        stat = torch.empty(shape[0], device="cuda")
        dw, db = torch.empty(n, 8, device="cuda"), torch.empty(n, device="cuda")
        short = ops.Checkpoint8(torch.empty(shape[0], 32, dtype=torch.int8, device="cuda"), torch.empty(shape[0], 1, dtype=torch.uint8, device="cuda"), 8)
        for call in (lambda: kept.store(x), lambda: kept.load(x), lambda: ops.ln_forward(x, gamma, gamma, y=x, mean=stat, rstd=stat),
                     lambda: ops.ln_backward(x, kept, None, stat, gamma, gamma, gamma, dx=x),
                     lambda: ops.CTensorApplyFunc.Backward(x, kept, x, "relu"), lambda: ops.checkpoint_wgrad(dw, db, x, short)):
            with pytest.raises(ops.B200Error, match="at most"):
                call()


def test_blocks_of_subnormal_numbers_keep_half_a_step_and_no_more():
    """Below 2^-126 the step stays 2^-132: off by 2^-133 at most, which for the smallest numbers is all of them."""
    x = np.zeros((3, 32), np.float32)
    x[0, 0], x[1, 3], x[2, :] = 2.0 ** -149, 2.0 ** -133, np.float32(2.0 ** -126) * (np.arange(32, dtype=np.float32) / 32)
    codes, exponents = cu.encode(x)
    v = cu.decode(codes, exponents, 32)
    assert (exponents == 1).all() and not v[:2].any()
    assert (np.abs(v - x.astype(np.float64)) <= 2.0 ** -133).all()
