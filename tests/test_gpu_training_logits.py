"""Logits of many features: the loss adds nothing of its own to them.

Where every product and every partial sum fits 24 bits the tensor cores lose
nothing, so the logits are exact.  Elsewhere a running sum is cut towards zero
at each 16-deep step: by at most 2^-23 of the partial sum there, and the step's
own products, aligned to the largest of them or the sum, by as much again.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_training import DTYPES, FN, give_memory_back, rand  # noqa: E402,F401


@pytest.fixture(scope="module")
def tr():
    from helrm_b200 import training
    return training


def wanted(l, t):
    """(loss, bound) for exact logits l: the sum of exponentials and its logarithm add FN, the two additions that make
    the loss half a unit in the last place of what they add up."""
    lse = torch.logsumexp(l, 1)
    at = l.gather(1, t[:, None])[:, 0]
    top = l.max(1).values
    return lse - at, 2 * FN + 2.0 ** -23 * ((top - at).abs() + (lse - at).abs())


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("inner", [64, 100, 512, 2048, 4096, 4100])
def test_exact_logits_stay_exact(tr, inner, dt):
    dt = DTYPES[dt]
    gen = torch.Generator(device="cuda").manual_seed(inner)
    n, v = 40, 300
    # one feature a row, the first a large one: a logit of 1024 beside others of 0
    h = torch.zeros(n, inner, device="cuda", dtype=dt)
    h[torch.arange(n), torch.randint(0, inner, (n,), generator=gen, device="cuda")] = 32
    w = torch.zeros(v, inner, device="cuda", dtype=dt)
    w[0] = 32
    w[1] = 29
    t = torch.arange(n, device="cuda") % 7
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    want, tol = wanted(h.double() @ w.double().T, t)
    assert ((loss.double() - want).abs() <= tol).all()
    assert (lse[:, 0] == 1024).all()
    # small whole numbers in every feature
    h = torch.randint(-2, 3, (n, inner), generator=gen, device="cuda").to(dt)
    w = torch.randint(-2, 3, (v, inner), generator=gen, device="cuda").to(dt)
    l = h.double() @ w.double().T
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    want, tol = wanted(l, t)
    assert (lse[:, 0].double() == l.max(1).values).all()
    assert ((loss.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("more", [1024, 4096])
def test_features_of_zeros_change_nothing(tr, more, dt):
    dt = DTYPES[dt]
    for inner in (24, 512):
        h, w = rand(130, inner, dtype=dt), rand(1000, inner, dtype=dt, std=2 * inner ** -0.5, seed=1)
        t = torch.arange(130, device="cuda") * 7
        ref = tr.vocabulary_loss_forward(h, w, t)
        pad = (0, more - inner)
        got = tr.vocabulary_loss_forward(torch.nn.functional.pad(h, pad), torch.nn.functional.pad(w, pad), t)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("inner", [512, 2048, 4096])
def test_dense_logits(tr, inner, dt):
    dt = DTYPES[dt]
    n, v = 64, 1000
    h, w = rand(n, inner, dtype=dt), rand(v, inner, dtype=dt, std=4 * inner ** -0.5, seed=1)
    t = torch.arange(n, device="cuda") * 3
    lost, total, part = (torch.zeros(n, v, dtype=torch.float64, device="cuda") for _ in range(3))
    for k in range(0, inner, 16):
        a, b = h[:, k:k + 16].double(), w[:, k:k + 16].double()
        before, part = part, part + a @ b.T
        lost += 2 * 2.0 ** -23 * torch.maximum(torch.maximum(before.abs(), part.abs()), a.abs() @ b.abs().T)
        if k % 1024 == 1008:
            total, part = total + part, torch.zeros_like(part)
            lost += 2.0 ** -24 * total.abs()
    total = total + part
    loss, _ = tr.vocabulary_loss_forward(h, w, t)
    want, tol = wanted(total, t)
    tol = tol + lost.max(1).values + lost.gather(1, t[:, None])[:, 0]
    assert ((loss.double() - want).abs() <= tol).all()
