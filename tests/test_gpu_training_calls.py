"""The training operators' calls at their edges, on a B200."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_training import DTYPES, block, give_memory_back  # noqa: E402,F401


@pytest.fixture(scope="module")
def tr():
    from helrm_b200 import training
    return training


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_an_empty_batch_of_a_frozen_block(tr, dt):
    """No tokens, and the input's gradient alone is wanted: it is empty."""
    dt = DTYPES[dt]
    _, wg, wu, _ = block((1, 40, 24), dt)
    x, dh = torch.empty(0, 40, device="cuda", dtype=dt), torch.empty(0, 24, device="cuda", dtype=dt)
    for kept in (x, tr.pack_checkpoint(x)):
        dx, dwg, dwu = tr.gated_backward(dh, kept, wg, wu, needs=(True, False, False))
        assert dx.shape == (0, 40) and dwg is None and dwu is None
    t = torch.empty(0, device="cuda", dtype=torch.int64)
    loss, lse = tr.vocabulary_loss_forward(x, wg, t)
    for w in (wg, torch.empty(30000, 40, device="cuda", dtype=dt), torch.empty(300, 100, device="cuda", dtype=dt)):
        h = torch.empty(0, w.shape[1], device="cuda", dtype=dt)
        dh, dw = tr.vocabulary_loss_backward(loss, h, w, t, lse, needs=(True, False))
        assert dh.shape == h.shape and dw is None
    x.requires_grad_()
    tr.gated_feed_forward(x, wg, wu).sum().backward()
    assert x.grad.shape == (0, 40)


def post(code):
    from helrm_b200 import _capi
    return _capi.load().helrm_TrainingPostFailure(0, code)


def test_a_kernel_that_gave_up_is_reported_once(tr):
    """By the next call or, after the last one, by synchronize.  The host leaves the word that the kernel would."""
    x, wg, wu, dh = block((10, 40, 24), torch.bfloat16)
    t = torch.zeros(10, dtype=torch.int64, device="cuda")
    tr.synchronize()
    loss, lse = tr.vocabulary_loss_forward(x, wg, t)
    c = tr.pack_checkpoint(x)
    for call in (lambda: tr.gated_forward(x, wg, wu), lambda: tr.gated_backward(dh, x, wg, wu),
                 lambda: tr.pack_checkpoint(x), lambda: tr.unpack_checkpoint(c),
                 lambda: tr.vocabulary_loss_forward(x, wg, t), lambda: tr.vocabulary_loss_backward(loss, x, wg, t, lse),
                 tr.synchronize, lambda: tr.synchronize(0), lambda: tr.synchronize("cuda:0")):
        assert post(4) == 0
        with pytest.raises(RuntimeError, match="gave up waiting .*code 4"):
            call()
        call()
        tr.synchronize()
    assert post(0) == -1 and post(-1) == -1
    tr.synchronize()


def test_synchronize_waits_for_its_stream(tr):
    x, wg, wu, _ = block((4096, 1024, 2048), torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(50):
            tr.gated_forward(x, wg, wu)
        done = s.record_event()
        tr.synchronize()
        assert done.query()


def test_transforms_without_a_rule_are_refused(tr):
    """Forward-mode derivatives and vmap have no rule here: they raise, and nothing comes back without its tangent."""
    x, wg, wu, _ = block((10, 40, 24), torch.bfloat16)
    w = torch.zeros(30, 24, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(10, dtype=torch.int64, device="cuda")
    h = tr.gated_forward(x, wg, wu)
    for f, a in ((lambda v: tr.gated_feed_forward(v, wg, wu), x), (lambda v: tr.gated_feed_forward(v, wg, wu, checkpoint=True), x),
                 (lambda v: tr.vocabulary_cross_entropy(v, w, t), h)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (a,), (torch.ones_like(a),))
    for f, a in ((lambda v: tr.gated_feed_forward(v, wg, wu), x), (lambda v: tr.vocabulary_cross_entropy(v, w, t[:1]), h)):
        with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
            torch.func.vmap(f)(a[:, None])
    # once differentiable: a second derivative raises
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(tr.gated_feed_forward(leaf, wg, wu).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaf)
    torch.cuda.synchronize()


def test_statistics_on_any_boundary(tr):
    """lse and dloss as views that start at an odd element give the same gradients."""
    h = torch.randn(33, 40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(torch.bfloat16)
    w, t = h.repeat(3, 1), torch.arange(33, device="cuda")
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    want = tr.vocabulary_loss_backward(loss, h, w, t, lse)

    def odd(v):
        buf = torch.empty(v.numel() + 1, device="cuda")
        buf[1:] = v.reshape(-1)
        return buf[1:].view(v.shape)
    for _ in range(2):
        got = tr.vocabulary_loss_backward(odd(loss), h, w, t, odd(lse))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
