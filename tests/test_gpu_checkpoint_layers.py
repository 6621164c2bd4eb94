"""Layers that normalise per sample and layers that keep what they need in 8 bits, run together as a net trains them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests import ckpt8_util as cu  # noqa: E402


@pytest.fixture(autouse=True)
def ops():
    from cuda_cnn_gan_vae_b200 import ops as o
    yield o
    o.set_precision(o.TF32X3)


def dense(batch, checkpoint8, share=True, widths=(96, 130, 64), inputs=200, func="leaky_relu"):
    from cuda_cnn_gan_vae_b200.layers import Net, NetLayerFunction, NetLayerLayerNormalization, NetLayerLinear
    spec = []
    for w in widths:
        spec += [(NetLayerLinear, dict(neurons=w)), (NetLayerLayerNormalization, {}), (NetLayerFunction, dict(func=func, leaky_slope=0.2))]
    spec.append((NetLayerLinear, dict(neurons=7)))
    keep = Net.share_tensors
    if not share:
        Net.share_tensors = lambda self: None
    try:
        return Net((1, inputs, 1), batch, spec, seed=1, checkpoint8=checkpoint8)
    finally:
        Net.share_tensors = keep


def rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


def wide_dense(net, x, error, slope=0.2, kept=None):
    """Gradients of sum(error * net(x)) in 64 bits by torch's autograd; kept: a list that receives what each layer reads."""
    from cuda_cnn_gan_vae_b200.layers import NetLayerFunction, NetLayerLayerNormalization, NetLayerLinear
    params = [{k: v.detach().double().requires_grad_() for k, v in layer.w.items()} if layer.param_shapes() else {} for layer in net.layers]
    x = x.double().reshape(net.batch, -1).requires_grad_()
    y = x
    for layer, w in zip(net.layers, params):
        if isinstance(layer, NetLayerLinear):
            y = y @ w["w"].view(layer.neurons, -1).t() + w["b"].view(-1)
        elif isinstance(layer, NetLayerLayerNormalization):
            mu = y.mean(1, keepdim=True)
            y = (y - mu) / ((y - mu).square().mean(1, keepdim=True) + layer.eps).sqrt() * w["gamma"].view(-1) + w["beta"].view(-1)
        elif isinstance(layer, NetLayerFunction):
            y = torch.where(y >= 0, y, slope * y)
    (y * error.double().reshape(net.batch, -1)).sum().backward()
    return y, x.grad, [{k: v.grad for k, v in w.items()} for w in params]


@pytest.mark.parametrize("batch", [1, 5, 64])
def test_net_with_layer_normalisation_against_autograd(ops, batch):
    """Without checkpoints: 3xTF32 products are off by about 2^-21 of their terms, each layer's gradient by a few of those."""
    net = dense(batch, False)
    x, error = torch.randn(batch, 1, 200, 1, device="cuda"), torch.randn(batch, 1, 7, 1, device="cuda")
    net.TrainingResetDeltaWeight()
    y = net.Forward(x)
    dx = net.TrainingBackward(error, True, need_input_error=True)
    ops.stream_status()
    want_y, want_dx, want = wide_dense(net, x, error)
    assert rel(y.view(batch, -1), want_y) < 1e-4
    assert rel(dx.view(batch, -1), want_dx) < 1e-4
    for layer, w in zip(net.layers, want):
        for name, g in w.items():
            assert rel(layer.g[name].view(-1), g.view(-1)) < 1e-4, name


@pytest.mark.parametrize("func", ["leaky_relu", "tanh", "sigmoid"])
@pytest.mark.parametrize("batch", [1, 5, 64])
def test_net_with_checkpoints(ops, batch, func):
    """The forward pass is that of the net without checkpoints, bit for bit.  A kept value is off by at most 1/127 of its block's
    largest, a normal one's rms by about 1 % of the tensor's; errors and gradients pass through three such tensors of
    each kind on their way, so 2-norms within 10 %, and not equal."""
    plain, kept = dense(batch, False, func=func), dense(batch, True, func=func)
    x, error = torch.randn(batch, 1, 200, 1, device="cuda"), torch.randn(batch, 1, 7, 1, device="cuda")
    outs = []
    for net in (plain, kept):
        net.TrainingResetDeltaWeight()
        outs.append((net.Forward(x).clone(), net.TrainingBackward(error, True, need_input_error=True).clone()))
    ops.stream_status()
    assert torch.equal(outs[0][0], outs[1][0])
    assert 0 < rel(outs[1][1], outs[0][1]) < 0.1
    for a, b in zip(plain.layers, kept.layers):
        for name in a.param_shapes():
            assert rel(b.g[name], a.g[name]) < 0.1, name
    # the last layer's bias gradient reads no kept value at all
    assert rel(kept.layers[-1].g["b"], plain.layers[-1].g["b"]) < 1e-6


def test_shared_tensors_change_nothing_and_inputs_may_go(ops):
    """Two output and two error tensors for the whole net: the same bits as tensors for every layer; and the net's input may be
    overwritten once Forward has returned."""
    apart, shared = dense(33, True, share=False), dense(33, True)
    assert len({layer.H.data_ptr() for layer in shared.layers}) == 2 and len({layer.H.data_ptr() for layer in apart.layers}) == 10
    x, error = torch.randn(33, 1, 200, 1, device="cuda"), torch.randn(33, 1, 7, 1, device="cuda")
    for turn in range(2):
        outs = []
        for net in (apart, shared):
            inp = x.clone()
            net.TrainingResetDeltaWeight()
            y = net.Forward(inp).clone()
            inp.fill_(float("nan"))
            dx = net.TrainingBackward(error, True, need_input_error=True).clone()
            outs.append((y, dx, net.grads.buffer.clone()))
        for a, b in zip(*outs):
            assert torch.equal(a, b) and torch.isfinite(a).all()
        x = x * 1.5
    # 33 bytes for 32 values
    layer = shared.layers[3]
    assert layer.kept.codes.numel() + layer.kept.exponents.numel() <= 33 * (96 * 33 // 32)


def test_function_layer_with_kept_signs_is_exact(ops):
    from cuda_cnn_gan_vae_b200.layers import NetLayerFunction
    for func in ("relu", "leaky_relu"):
        a, b = NetLayerFunction((3, 9, 11), 4, func), NetLayerFunction((3, 9, 11), 4, func, checkpoint8=True)
        x, e = torch.randn(4, 3, 9, 11, device="cuda"), torch.randn(4, 3, 9, 11, device="cuda")
        x[0] *= 1e-7
        assert torch.equal(a.Forward(x), b.Forward(x))
        assert torch.equal(a.TrainingBackward(e), b.TrainingBackward(e))


@pytest.mark.parametrize("dims", [1, 2, 3])
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_layer_normalisation_dims(ops, dims, checkpoint8):
    from cuda_cnn_gan_vae_b200.dp import GradArena
    from cuda_cnn_gan_vae_b200.layers import NetLayerLayerNormalization
    layer = NetLayerLayerNormalization((3, 10, 12), 4, dims=dims, checkpoint8=checkpoint8)
    w, g = GradArena(layer.param_shapes(), "cuda"), GradArena(layer.param_shapes(), "cuda")
    layer.bind(w.views, g.views)
    r = np.random.default_rng(dims)
    for v in w.views.values():
        v.copy_(torch.from_numpy(r.normal(1, 0.2, tuple(v.shape)).astype(np.float32)))
    g.buffer.zero_()
    x = torch.from_numpy(r.normal(1, 2, (4, 3, 10, 12)).astype(np.float32)).cuda()
    d = torch.from_numpy(r.normal(0, 1, (4, 3, 10, 12)).astype(np.float32)).cuda()
    y, dx = layer.Forward(x), layer.TrainingBackward(d)
    ops.stream_status()
    axes = tuple(range(4 - dims, 4))
    X, D = x.double().requires_grad_(), d.double()
    G, B = (w.views[k].double().requires_grad_() for k in ("gamma", "beta"))
    mu = X.mean(axes, keepdim=True)
    Y = (X - mu) / ((X - mu).square().mean(axes, keepdim=True) + 1e-6).sqrt() * G + B
    (Y * D).sum().backward()
    tol = 0.03 if checkpoint8 else 1e-5
    assert rel(y, Y) < 1e-6 and rel(dx, X.grad) < tol and rel(g.views["gamma"], G.grad) < tol and rel(g.views["beta"], B.grad) < 1e-6


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_discriminator_with_layer_normalisation(ops, checkpoint8):
    """Against autograd in 64 bits; and an image's answer does not depend on the rest of the batch."""
    from cuda_cnn_gan_vae_b200.nets import dcgan_discriminator
    net = dcgan_discriminator(4, image=(3, 32, 32), widths=(16, 32, 48), norm="layer", checkpoint8=checkpoint8)
    x = torch.randn(4, 3, 32, 32, device="cuda")
    net.TrainingResetDeltaWeight()
    y = net.Forward(x).clone()
    dx = net.TrainingBackward(torch.ones_like(y), True, need_input_error=True)
    ops.stream_status()
    X = x.double().requires_grad_()
    h, ws = X, []
    for i in range(3):
        conv, norm = net.layers[3 * i], net.layers[3 * i + 1]
        w = [conv.w["kernel"].double().requires_grad_(), conv.w["bias"].double().requires_grad_(), norm.w["gamma"].double().requires_grad_(),
             norm.w["beta"].double().requires_grad_()]
        ws.append((w, [conv.g["kernel"], conv.g["bias"], norm.g["gamma"], norm.g["beta"]]))
        h = torch.nn.functional.conv2d(h, w[0].view(conv.K, -1, 4, 4), w[1].view(-1), stride=2, padding=1)
        mu = h.mean((1, 2, 3), keepdim=True)
        h = (h - mu) / ((h - mu).square().mean((1, 2, 3), keepdim=True) + 1e-6).sqrt() * w[2] + w[3]
        h = torch.where(h >= 0, h, 0.2 * h)
    lin = net.layers[-2]
    w = [lin.w["w"].double().requires_grad_(), lin.w["b"].double().requires_grad_()]
    ws.append((w, [lin.g["w"], lin.g["b"]]))
    out = torch.sigmoid(h.reshape(4, -1) @ w[0].view(1, -1).t() + w[1].view(-1))
    out.sum().backward()
    assert rel(y.view(-1), out.view(-1)) < 1e-4
    # 3xTF32 convolutions without checkpoints; three kept tensors of each kind with them (as above)
    tol = 0.1 if checkpoint8 else 1e-3
    assert rel(dx, X.grad) < tol
    for want, got in ws:
        for a, b in zip(want, got):
            # (a convolution's bias in front of a normalisation shifts nothing but the few values at the borders' share: its
            # gradient is a difference of large sums, held to the size of what is summed)
            assert float((b.view(-1).double() - a.grad.view(-1)).norm()) <= tol * max(float(a.grad.norm()), 0.05 * float(dx.double().norm()))
    alone = net.Forward(torch.cat([x[:1], torch.randn(3, 3, 32, 32, device="cuda") * 3]))
    assert torch.equal(alone[0], y[0])


def test_vae_step_with_checkpointed_heads(ops):
    """The heads' forward passes and the errors they hand down are unchanged; their weight gradients come from the kept features."""
    from cuda_cnn_gan_vae_b200.nets import VAEStep
    grads = []
    x, eps = torch.rand(6, 3, 32, 32, device="cuda"), torch.randn(6, 1, 24, 1, device="cuda")
    for checkpoint8 in (False, True):
        step = VAEStep(6, image=(3, 32, 32), widths=(8, 16, 32), latent=24, checkpoint8=checkpoint8)
        x_hat = step(x, eps).clone()
        ops.stream_status()
        grads.append((x_hat, step.feat_error.clone(), step.mu.grads.buffer.clone(), step.logvar.grads.buffer.clone()))
    (h0, e0, m0, l0), (h1, e1, m1, l1) = grads
    assert torch.equal(h0, h1) and torch.equal(e0, e1)
    assert 0 < rel(m1, m0) < 0.03 and 0 < rel(l1, l0) < 0.03


@pytest.mark.parametrize("mode", ["TF32X3", "TF32", "FP32"])
def test_captured_training_steps(ops, mode):
    """Whole steps (forward, backward, Adam) captured and replayed give the weights of eager ones."""
    from cuda_cnn_gan_vae_b200.layers import AdamCorrections
    ops.set_precision(getattr(ops, mode))
    nets = [dense(40, True), dense(40, True)]
    x, error = torch.randn(40, 1, 200, 1, device="cuda"), torch.randn(40, 1, 7, 1, device="cuda")
    corr = AdamCorrections()

    def step(net):
        net.TrainingResetDeltaWeight()
        net.Forward(x)
        net.TrainingBackward(error)
        net.TrainingUpdateWeight(1e-3, None, corrections=corr.device)
    corr.set(1)
    step(nets[0]), step(nets[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(nets[1])
    for it in range(2, 5):
        corr.set(it)
        step(nets[0])
        graph.replay()
    ops.stream_status()
    assert torch.equal(nets[0].weights.buffer, nets[1].weights.buffer) and torch.isfinite(nets[0].weights.buffer).all()


def test_refusals(ops):
    from cuda_cnn_gan_vae_b200.layers import NetLayerLayerNormalization
    from cuda_cnn_gan_vae_b200.nets import dcgan_discriminator
    with pytest.raises(ops.B200Error):
        NetLayerLayerNormalization((3, 4, 5), 2, dims=4)
    with pytest.raises(ops.B200Error):
        dcgan_discriminator(2, image=(3, 32, 32), widths=(8,), norm="group")


FIRST_CALL = """
import sys
sys.path.insert(0, {root!r})
import torch
from cuda_cnn_gan_vae_b200 import ops
n = {n}
x, g, b = torch.randn(64, n, device="cuda"), torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
y, dx, mean, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
dg, db, delta = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.randn(64, 48, device="cuda")
dw, dbias, c = torch.empty(48, n, device="cuda"), torch.empty(48, device="cuda"), ops.Checkpoint8.empty(64, n)
def step():
    ops.ln_forward(x, g, b, y=y, mean=mean, rstd=rstd, checkpoint=c)
    ops.ln_backward(y, c, None, rstd, g, dg, db, accumulate=False, dx=dx)
    ops.CTensorApplyFunc.Backward(dx, c, dx, "tanh")
    ops.checkpoint_wgrad(dw, dbias, delta, c, accumulate=False)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (y, dx, dg, db, dw, dbias)]
step()
ops.stream_status()
assert all(torch.equal(a, b) for a, b in zip(got, (y, dx, dg, db, dw, dbias)))
print("captured")
"""


@pytest.mark.parametrize("n", [300, 20000])
def test_first_calls_of_a_process_inside_a_capture(n):
    """Nothing that a first call sets up is forbidden while a stream is captured."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=root, n=n)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


def chain(spec, shape, batch, share=True, checkpoint8=True, **kw):
    """A net, with or without tensors shared by its layers."""
    from cuda_cnn_gan_vae_b200.layers import Net
    keep = Net.share_tensors
    if not share:
        Net.share_tensors = lambda self: None
    try:
        return Net(shape, batch, spec, seed=3, checkpoint8=checkpoint8, **kw)
    finally:
        Net.share_tensors = keep


@pytest.mark.parametrize("layers", [2, 3, 4, 5])
def test_a_net_may_be_fed_its_own_output(ops, layers):
    """The output handed back as the next input, the error at the input as the next one at the output, for nets of two to five layers
    that share their tensors: the same bits as with tensors for every layer."""
    from cuda_cnn_gan_vae_b200.layers import NetLayerFunction, NetLayerLayerNormalization, NetLayerLinear
    n = 160
    kinds = [(NetLayerLinear, dict(neurons=n)), (NetLayerLayerNormalization, {}), (NetLayerLinear, dict(neurons=n)),
             (NetLayerFunction, dict(func="tanh")), (NetLayerLinear, dict(neurons=n))]
    x, error = torch.randn(9, 1, n, 1, device="cuda"), torch.randn(9, 1, n, 1, device="cuda")
    results = []
    for share in (False, True):
        net = chain(kinds[:layers], (1, n, 1), 9, share)
        y = x.clone()
        outs = []
        for _ in range(3):
            y = net.Forward(y if share else y.clone())
            outs.append(y.clone())
        e = error.clone()
        for _ in range(3):
            net.TrainingResetDeltaWeight()
            e = net.TrainingBackward(e if share else e.clone(), True, need_input_error=True)
            outs += [e.clone(), net.grads.buffer.clone()]
        ops.stream_status()
        results.append(outs)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def mixed():
    """A chain of every kind of layer: convolutions keep their inputs, the others let theirs go (the time embedding hands the error on)."""
    from cuda_cnn_gan_vae_b200 import layers as l
    return [(l.NetLayerTimeEmbedding, {}), (l.NetLayerConvolution, dict(kernel_amount=8, kernel_size=3, stride=1, padding=1)),
            (l.NetLayerLayerNormalization, {}), (l.NetLayerFunction, dict(func="leaky_relu")), (l.NetLayerMaxPooling, dict(pooling=2)),
            (l.NetLayerTimeEmbedding, {}), (l.NetLayerBatchNormalization, {}), (l.NetLayerFunction, dict(func="tanh")), (l.NetLayerUpSampling, dict(factor=2)),
            (l.NetLayerBackConvolution, dict(kernel_amount=6, kernel_size=4, stride=2, padding=1)),
            (l.NetLayerBatchNormalizationFunction, dict(func="leaky_relu")), (l.NetLayerConvolution, dict(kernel_amount=4, kernel_size=3, stride=2, padding=1)),
            (l.NetLayerFunction, dict(func="sigmoid")), (l.NetLayerLinear, dict(neurons=50)), (l.NetLayerFunction, dict(func="gelu")),
            (l.NetLayerLayerNormalization, dict(dims=2)), (l.NetLayerLinear, dict(neurons=3))]


@pytest.mark.parametrize("start", range(5))
def test_shared_tensors_of_mixed_nets_change_nothing(ops, start):
    """Nets that begin with any of the first layers of the chain, two steps each: the same bits as with tensors for every layer."""
    spec = mixed()
    shape = (2, 12, 16) if start < 2 else (8, 12, 16)
    x, error = torch.randn(6, *shape, device="cuda"), torch.randn(6, 1, 3, 1, device="cuda")
    results = []
    for share in (False, True):
        net = chain(spec[start:], shape, 6, share)
        outs = []
        for turn in range(2):
            net.TrainingResetDeltaWeight()
            y = net.Forward(x * (1 + turn))
            dx = net.TrainingBackward(error, True, need_input_error=True)
            outs += [y.clone(), dx.clone(), net.grads.buffer.clone()]
        ops.stream_status()
        results.append(outs)
        if share:
            names = [n for layer in net.layers for n in ("H", "prev_error", "delta") if getattr(layer, n, None) is not None]
            assert len({getattr(layer, n).data_ptr() for layer in net.layers for n in ("H", "prev_error", "delta") if getattr(layer, n, None) is not None}) < len(names)
    for a, b in zip(*results):
        assert torch.equal(a, b) and torch.isfinite(a).all()


def held(make):
    """What a net's construction leaves allocated and the most it had meanwhile, in bytes."""
    import gc
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    net = make()
    return net, torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("norm", ["batch", "layer"])
def test_checkpoints_save_memory_in_a_discriminator(ops, norm):
    """Per stage of N values without checkpoints: three outputs and three errors, and xhat of the batch normalisation.  With: the
    convolution's input and two checkpoints of 33 bytes for 32 values; outputs and errors are the largest stage's, twice each."""
    from cuda_cnn_gan_vae_b200.nets import dcgan_discriminator
    net, plain, _ = held(lambda: dcgan_discriminator(64, norm=norm))
    values = [64 * int(np.prod(layer.out_shape)) * 4 for layer in net.layers[:-2:3]]
    net, with_checkpoints, most = held(lambda: dcgan_discriminator(64, norm=norm, checkpoint8=True))
    # saved: outputs of convolution and normalisation and three errors of every stage; held: the shared ones, the checkpoints
    saved, cost = 5 * sum(values), 4 * max(values) + (33 / 128) * (2 if norm == "layer" else 1) * sum(values)
    assert with_checkpoints < plain - 0.9 * (saved - cost)
    # nor is more than that needed while it is made, but for one layer's own tensors
    assert most < with_checkpoints + 4 * max(values)


def test_vae_step_keeps_its_features_once(ops):
    """One checkpoint for both heads, and the features' own tensor used again on the way back: less memory than without, and the
    gradients of every step are those of heads with checkpoints and tensors of their own."""
    from cuda_cnn_gan_vae_b200.nets import VAEStep
    args = dict(image=(3, 64, 64), widths=(8, 16, 64), latent=24)
    _, plain, _ = held(lambda: VAEStep(16, **args))
    step, with_checkpoints, _ = held(lambda: VAEStep(16, checkpoint8=True, **args))
    feat, weights = 16 * 64 * 8 * 8 * 4, 2 * 24 * 64 * 8 * 8 * 4         # (the heads' scratch for weight gradients goes too)
    assert with_checkpoints < plain - weights - 0.7 * feat
    x, eps = torch.rand(16, 3, 64, 64, device="cuda"), torch.randn(16, 1, 24, 1, device="cuda")
    apart = VAEStep(16, checkpoint8=True, **args)
    feat_shape = apart.encoder.out_shape
    for net in (apart.mu, apart.logvar):
        head = net.layers[0]
        head.kept, head.stores = ops.Checkpoint8.empty(16, head.n_in), True
        head.prev_error = torch.empty((16,) + feat_shape, device="cuda")
    for turn in range(3):
        outs = [s(x, eps).clone() for s in (step, apart)]
        ops.stream_status()
        assert torch.equal(*outs) and torch.equal(step.feat_error, apart.feat_error)
        for a, b in zip(step.nets, apart.nets):
            assert torch.equal(a.grads.buffer, b.grads.buffer) and torch.equal(a.weights.buffer, b.weights.buffer)


@pytest.mark.parametrize("norm,checkpoint8", [("layer", False), ("layer", True), ("batch", True)])
def test_dcgan_step_with_such_a_discriminator(ops, norm, checkpoint8):
    """Captured and replayed steps leave the weights that eager ones do."""
    from cuda_cnn_gan_vae_b200.nets import DCGANStep
    args = dict(widths_g=(32, 16, 8, 3), widths_d=(8, 16, 32, 48), base=64, norm=norm, checkpoint8=checkpoint8)
    z, labels = torch.randn(8, 1, 100, 1, device="cuda"), torch.ones(8, 1, 1, 1, device="cuda")
    steps = [DCGANStep(8, use_graph=g, **args) for g in (False, True)]
    assert (steps[0].D.layers[-1].kept is not None) == checkpoint8
    assert type(steps[0].D.layers[1]).__name__ == ("NetLayerLayerNormalization" if norm == "layer" else "NetLayerBatchNormalization")
    for _ in range(5):
        outs = [s(z, labels).clone() for s in steps]
        ops.stream_status()
        assert torch.equal(*outs)
    assert steps[1].graph is not None
    for a, b in zip((steps[0].G, steps[0].D), (steps[1].G, steps[1].D)):
        assert torch.equal(a.weights.buffer, b.weights.buffer) and torch.isfinite(a.weights.buffer).all()
