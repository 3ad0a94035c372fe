"""The training operators' ways through their kernels: each case is of a size
that takes a branch the others leave out.

Free blocks of torch's allocator hold NaN here, so that an output tile that no
block writes shows.  The narrow gradients' kernel is one of three launches of
its call; the pieces' way has four at least.
"""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_training import (ACC, DTYPES, V, block, gated_grads, give_memory_back, loss_grads, rand,  # noqa: E402,F401
                               within)


@pytest.fixture(scope="module")
def tr():
    from helrm_b200 import training
    return training


def spoil(n):
    """NaN in the blocks that the next allocations come from."""
    parts = [torch.full((m,), float("nan"), device="cuda") for m in (n, n, n, n)]
    torch.cuda.synchronize()
    del parts


def launches():
    from helrm_b200 import _capi
    n = ctypes.c_uint64(0)
    _capi.check(_capi.load().helrm_GetLaunchCount(ctypes.byref(n)))
    return n.value


# dX and the weights' gradients in one launch, (tokens, inner, width): clusters that the first one's last round leaves
# out take the second's tiles, which that round has room for (80 tiles in all), which it has not, after a whole round of
# the first's, and where the first one's rounds are all whole
TOGETHER = [(2047, 1001, 1500), (266, 263, 1829), (3000, 1100, 1300), (281, 9791, 265), (263, 9321, 217)]
# a launch each: 128 tiles of 8 tile rows, 160 of 20 (more than the 74 SM pairs take at once, in groups of 8 rows)
APART = [(2048, 2048, 2048), (1500, 1000, 5000)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", TOGETHER + APART)
def test_gated_gradients(tr, shape, dt):
    x, wg, wu, dh = block(shape, DTYPES[dt])
    spoil(max(x.numel(), wg.numel(), dh.numel()))
    got = tr.gated_backward(dh, x, wg, wu)
    for g, w, what in zip(got, gated_grads(dh, x, wg, wu, "silu"), ("dx", "dw_gate", "dw_up")):
        within(g, w, what)


def loss_case(shape, dt, ignored=0.0):
    n, k, v = shape
    h, w = rand(n, k, dtype=dt), rand(v, k, dtype=dt, std=2 * k ** -0.5, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(n + v)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    t[torch.rand(n, generator=gen, device="cuda") < ignored] = -100
    g = (0.5 + torch.rand(n, generator=gen, device="cuda")) * (1024.0 if dt == torch.float16 else 1.0) / n
    return h, w, t, g


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(204, 258, 4961), (281, 9791, 265), (272, 9706, 457), (260, 9395, 265),
                                   (777, 432, 32001)])
def test_loss_gradients(tr, shape, dt):
    h, w, t, g = loss_case(shape, DTYPES[dt])
    _, lse = tr.vocabulary_loss_forward(h, w, t)
    spoil(max(h.numel(), w.numel()))
    got = tr.vocabulary_loss_backward(g, h, w, t, lse)
    for a, want, what in zip(got, loss_grads(g, h, w, t), ("dh", "dw")):
        within(a, want, what)


# tokens x inner x vocab, with no row ignored: 128 / depth token tiles a group, depth the features in sixteens
GROUPS = [(3000, 16, 18944, 3), (4096, 9, 18944, 4), (1300, 32, 18944, 3), (1000, 40, 18944, 4), (1000, 48, 18900, 4),
          (700, 64, 18944, 3), (900, 50, 18930, 4)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", GROUPS)
def test_narrow_loss_gradients_in_groups(tr, shape, dt):
    """Three groups of token tiles and more at every depth: the middle ones add to what the first one wrote."""
    n, k, v, groups = shape
    depth = -(-k // 16) * 16
    assert -(-(-(-n // 128)) // (128 // depth)) == groups
    for ignored in (0.0, 0.1):
        h, w, t, g = loss_case((n, k, v), DTYPES[dt], ignored)
        keep = t != -100
        assert -(-(-(-int(keep.sum()) // 128)) // (128 // depth)) >= 3
        _, lse = tr.vocabulary_loss_forward(h, w, t)
        w = w if k % 8 == 0 else torch.nn.functional.pad(w, (0, -k % 8))[:, :k]  # rows that need no copy
        spoil(max(h.numel(), w.numel()))
        before = launches()
        dh, dw = tr.vocabulary_loss_backward(g, h, w, t, lse)
        assert launches() - before == 3  # gathering, the kernel, joining
        wdh, wdw = loss_grads(g[keep], h[keep], w, t[keep])
        within(dh[keep].contiguous(), wdh, "dh")
        within(dw, wdw, "dw")
        assert not dh[~keep].any()
