"""The loss's two passes form the same logits: a row that is certain of its
target, whose logit is about 1000 and 150 and more above all others, has a loss
of zero and no gradient (exp(-150) is no 32-bit number)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_training import DTYPES, give_memory_back, rand  # noqa: E402,F401


@pytest.fixture(scope="module")
def tr():
    from helrm_b200 import training
    return training


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(4, 16, 300), (4, 64, 300), (4, 16, 30000), (4, 64, 40000), (40, 100, 700),
                                   (300, 512, 1000), (300, 520, 1000), (300, 1024, 1000), (70, 2500, 900),
                                   (300, 4096, 5000)])
def test_certain_rows_have_no_gradient(tr, shape, dt):
    n, k, v = shape
    dt = DTYPES[dt]
    h = rand(n, k, dtype=dt)
    w = rand(v, k, dtype=dt, std=k ** -0.5, seed=1)
    t = torch.arange(n, device="cuda") * (v // n)
    w[t] = (h.float() * (1000 / h.float().square().sum(1, keepdim=True))).to(dt)
    l = h.double() @ w.double().T
    at = l.gather(1, t[:, None])
    sure = ((at - l) > 150).sum(1) == v - 1  # few features: another row's direction may be near
    assert int(sure.sum()) >= n // 2
    t = torch.where(sure, t, torch.full_like(t, -100))
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    assert not loss.any()
    dh, dw = tr.vocabulary_loss_backward(torch.ones(n, device="cuda"), h, w, t, lse)
    assert not dh.any() and not dw.any()
