"""What a refused call leaves behind: nothing."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_a_refused_launch_does_not_fail_the_next_call():
    """A launch that the runtime refuses on the host (a matrix of more rows than the transposition's grid has blocks for) is that
    call's error, and that one's only."""
    from cuda_cnn_gan_vae_b200 import ops
    from cuda_cnn_gan_vae_b200.lib import load
    rows = 32 * 65535 + 1
    a, b = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    refused = load().b200_transpose(b.data_ptr(), a.data_ptr(), 1, rows, 1, None)
    assert refused in (0, 3)
    x, gamma = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    ops.ln_forward(x, gamma, gamma)
    ops.Checkpoint8.empty(4, 64).store(x)
    ops.stream_status()
    torch.cuda.synchronize()
