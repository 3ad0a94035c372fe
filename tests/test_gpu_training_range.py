"""The gated block's gradients in half precision where dH times a projection
is outside that type's range and the gradients themselves are inside it.

dG and dU are rounded to 16 bits once, relative to a power of two that brings
a bound of both, B = max_i(max|dH_i| |x_i|) max(1.13 max|wu_j|, max|wg_j|)
(norms of rows), to at least 2^14: a subnormal step of half precision, 2^-24,
is then at most 2^-38 of B, and rounding to it half of that.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_training import (DTYPES, V, act, add, give_memory_back, mm, mul, tr_, unit, within)  # noqa: E402,F401


@pytest.fixture(scope="module")
def tr():
    from helrm_b200 import training
    return training


def normal(*shape, std, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def grads(dh, x, wg, wu, name):
    dt = dh.dtype
    b = 0.0
    if dt == torch.float16:
        tokens = (dh.double().abs().max(1).values * x.double().norm(dim=1)).max()
        b = float(tokens * torch.maximum(1.13 * wu.double().norm(dim=1).max(), wg.double().norm(dim=1).max()))

    def once(a):
        return V(a.v, a.e + unit(dt) * a.m + 2.0 ** -39 * 1.01 * b)
    x, wg, wu, dh = V(x), V(wg), V(wu), V(dh)
    a, d = act(mm(x, wg), name)
    dg = once(mul(mul(dh, mm(x, wu)), d))
    du = once(mul(dh, a))
    return add(mm(dg, tr_(wg)), mm(du, tr_(wu))), mm(tr_(dg), tr_(x)), mm(tr_(du), tr_(x))


def large(dt, shape=(64, 72, 96)):
    t, k, f = shape
    return (normal(t, f, std=4096, dtype=dt, seed=1), normal(t, k, std=0.02, dtype=dt, seed=2),
            normal(f, k, std=5e-3, dtype=dt, seed=3), normal(f, k, std=100, dtype=dt, seed=4))


def check(tr, dh, x, wg, wu, name):
    want = grads(dh, x, wg, wu, name)
    for v in want:  # the case is one whose gradients the type holds
        assert float(v.v.abs().max()) < 65000
    for got, w, what in zip(tr.gated_backward(dh, x, wg, wu, name), want, ("dx", "dw_gate", "dw_up")):
        within(got, w, what)


@pytest.mark.parametrize("name", ["identity", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_products_above_the_range(tr, dt, name):
    args = large(DTYPES[dt])
    assert float((args[0].double() * (args[1].double() @ args[3].double().T)).abs().max()) > 70000
    check(tr, *args, name)


@pytest.mark.parametrize("name", ["identity", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_products_below_the_range(tr, dt, name):
    dt = DTYPES[dt]
    t, k, f = 2048, 40, 72
    check(tr, normal(t, f, std=1e-5, dtype=dt, seed=1), normal(t, k, std=100, dtype=dt, seed=2),
          normal(f, k, std=2e-5, dtype=dt, seed=3), normal(f, k, std=2e-3, dtype=dt, seed=4), name)


def test_from_a_checkpoint_and_odd_rows(tr):
    """The same gradients whatever the rows' pitch, and from the 8-bit copy as from its values."""
    dh, x, wg, wu = large(torch.float16, (300, 71, 136))
    ref = tr.gated_backward(dh, x, wg, wu)

    def odd(t):
        buf = torch.zeros(t.shape[0], t.shape[1] + 5, dtype=t.dtype, device="cuda")
        buf[:, 3:3 + t.shape[1]] = t
        return buf[:, 3:3 + t.shape[1]]
    for a, b in zip(tr.gated_backward(odd(dh), odd(x), odd(wg), odd(wu)), ref):
        assert torch.equal(a, b)
    c = tr.pack_checkpoint(x)
    for a, b in zip(tr.gated_backward(dh, c, wg, wu), tr.gated_backward(dh, tr.unpack_checkpoint(c), wg, wu)):
        assert torch.equal(a, b)
    for i in range(3):
        one = tr.gated_backward(dh, x, wg, wu, needs=[j == i for j in range(3)])
        assert torch.equal(one[i], ref[i])


def test_one_token_that_is_not_finite(tr):
    """What one token holds does not change the range of the others."""
    dh, x, wg, wu = large(torch.float16)
    want = grads(dh, x, wg, wu, "silu")[0]
    keep = torch.arange(64, device="cuda") != 9
    for what in ("x", "dh"):
        for bad in (float("inf"), float("nan")):
            x2, dh2 = x.clone(), dh.clone()
            (x2 if what == "x" else dh2)[9, 5] = bad
            dx = tr.gated_backward(dh2, x2, wg, wu)[0]
            within(dx[keep], V(want.v[keep], want.e[keep]), what)
            assert not torch.isfinite(dx[9]).all()


def test_gradients_of_zero(tr):
    dh, x, wg, wu = large(torch.float16)
    for args in ((torch.zeros_like(dh), x, wg, wu), (dh, torch.zeros_like(x), wg, wu)):
        for g in tr.gated_backward(*args):
            assert torch.isfinite(g).all()
    dx, dwg, dwu = tr.gated_backward(torch.zeros_like(dh), x, wg, wu)
    assert not dx.any() and not dwg.any() and not dwu.any()


@pytest.mark.parametrize("shape", [(3, 5000, 40), (40, 64, 5000), (1, 1, 1), (700, 4100, 30)])
def test_long_rows(tr, shape):
    t, k, f = shape
    dt = torch.float16
    check(tr, normal(t, f, std=1000, dtype=dt, seed=1), normal(t, k, std=0.05, dtype=dt, seed=2),
          normal(f, k, std=0.01, dtype=dt, seed=3), normal(f, k, std=1.0, dtype=dt, seed=4), "silu")


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_outliers(tr, dt):
    """Tokens of large dH and tokens of long x, not the same ones: neither takes the others' bits."""
    dt = DTYPES[dt]
    t, k, f = 300, 512, 136
    dh, x = normal(t, f, std=1e-2, dtype=dt, seed=1), normal(t, k, std=0.5, dtype=dt, seed=2)
    wg, wu = normal(f, k, std=0.02, dtype=dt, seed=3), normal(f, k, std=0.02, dtype=dt, seed=4)
    dh[::50] = normal(6, f, std=2000, dtype=dt, seed=5)
    x[7::50, 3] = 2000.0
    for name in ("identity", "silu"):
        check(tr, dh, x, wg, wu, name)
