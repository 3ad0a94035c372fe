"""The training operators on a B200 against their formulas in 64 bits.

Tolerances are bounds carried along with the values: every 64-bit value has
an error bound beside it, a product of K terms adds K 2^-23 of the sum of the
terms' magnitudes (32-bit accumulation in any order, truncated or rounded),
a rounding to the 16-bit type adds half a unit in the last place (2^-8 for
bfloat16, 2^-11 for half precision, whose subnormals add 2^-25), and a
function adds its slope times the bound plus 2^-20 of its value for its own
evaluation.  Every element has to lie within its own bound.
"""
import gc
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def give_memory_back():
    """The tests after these find torch's allocator as if these had not run."""
    yield
    gc.collect()
    torch.cuda.empty_cache()


DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACC = 2.0 ** -23
FN = 2.0 ** -20


@pytest.fixture(scope="module")
def tr():
    from helrm_b200 import training
    return training


def unit(dtype):
    return torch.finfo(dtype).eps / 2


class V:
    """A 64-bit value and the bound of what the kernel's may differ by."""

    def __init__(self, v, e=None):
        self.v = v.double()
        self.e = torch.zeros_like(self.v) if e is None else e

    @property
    def m(self):
        return self.v.abs() + self.e


def mm(a, b):
    """a b^T"""
    return V(a.v @ b.v.T, a.e @ b.m.T + a.v.abs() @ b.e.T + a.v.shape[1] * ACC * (a.m @ b.m.T))


def tr_(a):
    return V(a.v.T, a.e.T)


def add(a, b):
    return V(a.v + b.v, a.e + b.e + ACC * (a.m + b.m))


def mul(a, b):
    return V(a.v * b.v, a.e * b.m + a.v.abs() * b.e + ACC * a.m * b.m)


def rnd(a, dtype):
    return V(a.v, a.e + unit(dtype) * a.m + (2.0 ** -25 if dtype == torch.float16 else 0.0))


def act(g, name):
    """(act(g), act'(g))"""
    x = g.v
    if name == "identity":
        return g, V(torch.ones_like(x))
    if name == "relu":
        near = (x.abs() <= g.e).double()  # the sign may be the other one
        return V(x.clamp(min=0), g.e), V((x > 0).double(), near)
    if name == "silu":
        s = torch.sigmoid(x)
        a, d = x * s, s * (1 + x * (1 - s))
        # |silu'| <= 1.1, |silu''| <= 0.5
        return V(a, 1.1 * g.e + FN * (a.abs() + g.e)), V(d, 0.5 * g.e + FN * (1 + x.abs()))
    s = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    p = torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    a, d = x * s, s + x * p
    # |gelu'| <= 1.13, |gelu''| <= 0.8; Phi carries 2^-20 of 1, not of its value
    return V(a, 1.13 * g.e + FN * x.abs()), V(d, 0.8 * g.e + FN * (1 + x.abs()))


def gated(x, wg, wu, name):
    return mul(act(mm(V(x), V(wg)), name)[0], mm(V(x), V(wu)))


def gated_grads(dh, x, wg, wu, name):
    dt = dh.dtype
    x, wg, wu, dh = V(x), V(wg), V(wu), V(dh)
    a, d = act(mm(x, wg), name)
    dg = rnd(mul(mul(dh, mm(x, wu)), d), dt)
    du = rnd(mul(dh, a), dt)
    return add(mm(dg, tr_(wg)), mm(du, tr_(wu))), mm(tr_(dg), tr_(x)), mm(tr_(du), tr_(x))


def within(got, want, what=""):
    """got is the 16-bit (or 32-bit) result of want's value."""
    w = rnd(want, got.dtype) if got.dtype != torch.float32 else V(want.v, want.e + 2.0 ** -24 * want.m)
    assert got.shape == w.v.shape, what
    off = (got.double() - w.v).abs()
    assert torch.isfinite(got).all(), what
    over = off > w.e
    assert not over.any(), f"{what}: {int(over.sum())} of {over.numel()} elements over their bound, the worst by a factor " \
                           f"{float((off / w.e.clamp(min=1e-300)).max()):.3g}"


def rand(*shape, dtype, std=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum((i + 1) * s for i, s in enumerate(shape)))
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


SHAPES = [(1, 1, 1), (1, 64, 8), (2, 13, 512), (5, 16, 33), (64, 432, 512), (127, 8, 129), (128, 256, 128),
          (129, 100, 257), (256, 64, 256), (257, 72, 130), (300, 520, 71), (1000, 24, 40), (33, 2100, 19),
          (513, 136, 640)]


def block(shape, dtype):
    t, k, f = shape
    return (rand(t, k, dtype=dtype), rand(f, k, dtype=dtype, std=k ** -0.5, seed=1),
            rand(f, k, dtype=dtype, std=k ** -0.5, seed=2), rand(t, f, dtype=dtype, seed=3))


@pytest.mark.parametrize("name", ["identity", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gated(tr, shape, dt, name):
    x, wg, wu, dh = block(shape, DTYPES[dt])
    within(tr.gated_forward(x, wg, wu, name), gated(x, wg, wu, name), "h")
    for got, want, what in zip(tr.gated_backward(dh, x, wg, wu, name), gated_grads(dh, x, wg, wu, name),
                               ("dx", "dw_gate", "dw_up")):
        within(got, want, what)


def test_gated_extremes(tr):
    """Gates far from zero: the activation saturates and nothing overflows on the way."""
    x = torch.tensor([[1.0], [-1.0], [0.0], [-0.0]], device="cuda", dtype=torch.bfloat16)
    wg = torch.tensor([[1e4], [-1e4], [300.0], [88.0], [1e38]], device="cuda", dtype=torch.bfloat16)
    wu = torch.ones_like(wg)
    for name in ("silu", "gelu", "relu"):
        h = tr.gated_forward(x, wg, wu, name).double()
        g = x.double() @ wg.double().T
        want = g.clamp(min=0) * x.double()
        assert torch.allclose(h, want, rtol=2.0 ** -8, atol=1e-30), name
        dx, dwg, dwu = tr.gated_backward(torch.ones(4, 4, device="cuda", dtype=x.dtype), x, wg[:4], wu[:4], name)
        assert all(torch.isfinite(t).all() for t in (dx, dwg, dwu)), name


def test_gated_passes_on_what_is_not_finite(tr):
    x, wg, wu, _ = block((40, 48, 24), torch.bfloat16)
    x = x.clone()
    x[7, 3] = float("nan")
    for name in ("identity", "relu", "silu", "gelu"):
        h = tr.gated_forward(x, wg, wu, name)
        assert torch.isnan(h[7]).all() and torch.isfinite(h[:7]).all() and torch.isfinite(h[8:]).all()


def placed(t, how):
    """t with other strides and alignments."""
    rows, cols = t.shape
    if how == "odd":  # an odd row pitch, rows that start at odd elements
        buf = torch.zeros(rows, cols + 5, dtype=t.dtype, device=t.device)
        buf[:, 3:3 + cols] = t
        return buf[:, 3:3 + cols]
    if how == "wide":  # a pitch that vector loads fit, more than the columns
        buf = torch.zeros(rows, cols + 64 + -cols % 8, dtype=t.dtype, device=t.device)
        buf[:, 8:8 + cols] = t
        return buf[:, 8:8 + cols]
    return t.T.contiguous().T  # columns first


@pytest.mark.parametrize("how", ["odd", "wide", "columns"])
def test_strides(tr, how):
    for dt in DTYPES.values():
        x, wg, wu, dh = block((150, 72, 136), dt)
        ref = (tr.gated_forward(x, wg, wu), *tr.gated_backward(dh, x, wg, wu))
        a = [placed(t, how) for t in (x, wg, wu, dh)]
        assert not a[0].is_contiguous()
        got = (tr.gated_forward(*a[:3]), *tr.gated_backward(a[3], *a[:3]))
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
        w = rand(500, 72, dtype=dt, std=0.2, seed=5)
        t = torch.arange(150, device="cuda") * 3
        loss, lse = tr.vocabulary_loss_forward(x, w, t)
        g = torch.rand(150, device="cuda")
        ref = (loss, lse, *tr.vocabulary_loss_backward(g, x, w, t, lse))
        wp = placed(w, how)
        t2 = torch.stack([t, t], 1)[:, 0].to(torch.int32)
        loss, lse = tr.vocabulary_loss_forward(a[0], wp, t2)
        got = (loss, lse, *tr.vocabulary_loss_backward(torch.stack([g, g], 1)[:, 1], a[0], wp, t2, lse))
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
        c, r = tr.pack_checkpoint(a[0]), tr.pack_checkpoint(x)
        assert torch.equal(c.q, r.q) and torch.equal(c.e, r.e)


def test_leading_dimensions(tr):
    x, wg, wu, dh = block((60, 40, 24), torch.bfloat16)
    x3, dh3 = x.view(3, 4, 5, 40), dh.view(3, 4, 5, 24)
    assert torch.equal(tr.gated_forward(x3, wg, wu).view(60, 24), tr.gated_forward(x, wg, wu))
    for a, b in zip(tr.gated_backward(dh3, x3, wg, wu), tr.gated_backward(dh, x, wg, wu)):
        assert torch.equal(a.reshape(b.shape), b)
    one = tr.gated_forward(x[0], wg, wu)
    assert one.shape == (24,) and torch.equal(one, tr.gated_forward(x[:1], wg, wu)[0])
    c = tr.pack_checkpoint(x3)
    assert c.shape == x3.shape and tr.unpack_checkpoint(c).shape == x3.shape
    # an expanded input: rows that share memory
    xe = x[:1].expand(7, 40)
    assert torch.equal(tr.gated_forward(xe, wg, wu), tr.gated_forward(x[:1], wg, wu).expand(7, 24))


def test_needs(tr):
    x, wg, wu, dh = block((70, 40, 24), torch.float16)
    full = tr.gated_backward(dh, x, wg, wu)
    for i in range(3):
        needs = [j == i for j in range(3)]
        got = tr.gated_backward(dh, x, wg, wu, needs=needs)
        assert [g is None for g in got] == [not n for n in needs] and torch.equal(got[i], full[i])
    assert tr.gated_backward(dh, x, wg, wu, needs=(False, False, False)) == (None, None, None)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_no_tokens(tr, dt):
    dt = DTYPES[dt]
    _, wg, wu, _ = block((1, 40, 24), dt)
    x, dh = torch.empty(0, 40, device="cuda", dtype=dt), torch.empty(0, 24, device="cuda", dtype=dt)
    assert tr.gated_forward(x, wg, wu).shape == (0, 24)
    dx, dwg, dwu = tr.gated_backward(dh, x, wg, wu)
    assert dx.shape == (0, 40) and not dwg.any() and not dwu.any() and dwg.shape == wg.shape
    c = tr.pack_checkpoint(x)
    assert tr.unpack_checkpoint(c).shape == (0, 40)
    dx, dwg, dwu = tr.gated_backward(dh, c, wg, wu)
    assert dx.shape == (0, 40) and not dwg.any() and not dwu.any()
    t = torch.empty(0, device="cuda", dtype=torch.int64)
    loss, lse = tr.vocabulary_loss_forward(x, wg, t)
    assert loss.shape == (0,) and lse.shape == (0, 2)
    d, dw = tr.vocabulary_loss_backward(loss, x, wg, t, lse)
    assert d.shape == (0, 40) and dw.shape == wg.shape and not dw.any()


# ------------------------------------------------------------------ checkpoints
def checkpoint_values(x):
    """The values of the definition, in 64 bits: for each group the least
    power of two s (within the type's range) with max |x| <= 127 s."""
    half = x.dtype == torch.float16
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=torch.float64)
    xs = x.double().cpu()
    for r in range(rows):
        for c in range(0, cols, 32):
            g = xs[r, c:c + 32]
            if not torch.isfinite(g).all():
                out[r, c:c + 32] = math.nan
                continue
            e = -24 if half else -126
            top = float(g.abs().max())
            while top > 127 * 2.0 ** e:
                e += 1
            lim = math.floor(torch.finfo(x.dtype).max / 2.0 ** e)
            for i, v in enumerate(g.tolist()):
                out[r, c + i] = max(-lim, min(lim, round(v / 2.0 ** e))) * 2.0 ** e  # round(): halves to even
    return out


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (4, 32), (5, 33), (7, 100), (9, 13), (2, 1000), (33, 64)])
def test_checkpoint_is_its_definition(tr, dt, shape):
    x = rand(*shape, dtype=DTYPES[dt])
    x = x * (10.0 ** torch.randint(-3, 3, (shape[0], 1), device="cuda")).to(x.dtype)
    c = tr.pack_checkpoint(x)
    assert torch.equal(tr.unpack_checkpoint(c).double().cpu(), checkpoint_values(x))
    groups = -(-shape[1] // 32)
    assert c.q.shape == (shape[0], 32 * groups) and not c.q[:, shape[1]:].any()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_checkpoint_edges(tr, dt):
    dt = DTYPES[dt]
    f = torch.finfo(dt)
    x = torch.zeros(12, 32, dtype=dt, device="cuda")
    x[1, 5] = f.max
    x[2, :] = torch.linspace(-1, 1, 32).to(dt) * f.max
    x[3, 0] = f.smallest_subnormal if hasattr(f, "smallest_subnormal") else f.tiny
    x[4, 0] = f.tiny
    x[5, 0], x[5, 1] = float("inf"), 1.0
    x[6, 0], x[6, 1] = float("nan"), 1.0
    x[7, 0], x[7, 1] = float("-inf"), 1.0
    x[8, 0], x[8, 1], x[8, 2], x[8, 3] = 127.0, 0.5, 1.5, 2.5   # s = 1: halves to even
    x[9, 0], x[9, 1] = 127.5, 1.0                                # s = 2
    x[10, 0], x[10, 1] = -128.0, 3.0
    x[11, :] = -f.max
    got, want = tr.unpack_checkpoint(tr.pack_checkpoint(x)).double().cpu(), checkpoint_values(x)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.isnan(want).sum() == 3 * 32
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_checkpoint_long(tr):
    x = rand(70001, 264, dtype=torch.bfloat16)
    got = tr.unpack_checkpoint(tr.pack_checkpoint(x))
    s = x.float().view(70001, -1)
    for a, b in ((0, 32), (224, 256), (256, 264)):
        assert ((got[:, a:b].float() - s[:, a:b]).abs() <= s[:, a:b].abs().amax(1, keepdim=True) / 127).all()
    rows = torch.tensor([0, 1, 35000, 69999, 70000], device="cuda")
    assert torch.equal(got[rows].double().cpu(), checkpoint_values(x[rows]))


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 13, 8), (64, 432, 512), (129, 100, 257), (300, 40, 71)])
def test_backward_from_checkpoint(tr, dt, shape):
    x, wg, wu, dh = block(shape, DTYPES[dt])
    c = tr.pack_checkpoint(x)
    got = tr.gated_backward(dh, c, wg, wu, "gelu")
    for g, w, what in zip(got, gated_grads(dh, tr.unpack_checkpoint(c), wg, wu, "gelu"), ("dx", "dw_gate", "dw_up")):
        within(g, w, what)
    # the same bits as from the values read back
    for g, w in zip(got, tr.gated_backward(dh, tr.unpack_checkpoint(c), wg, wu, "gelu")):
        assert torch.equal(g, w)


# ------------------------------------------------------------------ the loss
def loss_values(h, w, t, ignore=-100):
    l = mm(V(h), V(w))
    lse = torch.logsumexp(l.v, 1)
    valid = t != ignore
    tt = torch.where(valid, t.long(), torch.zeros_like(t.long()))[:, None]
    # lse moves by at most the largest bound of its row's logits; exp and log add FN (the terms' exponents are of
    # order |l - max|, rounded once)
    e = l.e.max(1).values + FN * (1 + (l.v - l.v.max(1, keepdim=True).values).abs().clamp(max=30).max(1).values * 0.25
                                  + lse.abs())
    loss = torch.where(valid, lse - l.v.gather(1, tt)[:, 0], torch.zeros_like(lse))
    return l, V(lse, e), V(loss, torch.where(valid, e + l.e.gather(1, tt)[:, 0], torch.zeros_like(e))), valid, tt


def loss_grads(g, h, w, t, ignore=-100):
    l, lse, _, valid, tt = loss_values(h, w, t, ignore)
    arg = l.v - lse.v[:, None]
    p = torch.exp(arg)
    ep = p * (torch.expm1(l.e + lse.e[:, None]) + FN * (1 + 0.25 * arg.abs()))
    hot = torch.zeros_like(p).scatter_(1, tt, 1.0)
    gg = torch.where(valid, g.double(), torch.zeros_like(g.double()))[:, None]
    z, ez = (p - hot) * gg, ep * gg.abs()
    # Z in the 16-bit type; half precision scales it by a power of two first, to at least 2^-39 of the largest row's
    ez = ez + unit(h.dtype) * (z.abs() + ez)
    if h.dtype == torch.float16:
        ez = ez + 2.0 ** -39 * gg.abs().max()
    z = V(z, ez)
    return mm(z, tr_(V(w))), mm(tr_(z), tr_(V(h)))


LOSSES = [(1, 1, 1), (1, 16, 3), (2, 13, 1000), (64, 64, 1000), (127, 8, 129), (128, 256, 256), (129, 100, 257),
          (300, 432, 5003), (777, 24, 2049), (256, 16, 40001), (33, 1025, 130)]


# narrow rows over a vocabulary of every block's share: one token tile and several groups of them, every depth
NARROW = [(64, 3, 30000), (1, 16, 19000), (1025, 16, 20001), (1000, 24, 18944), (130, 64, 19457), (2000, 50, 19001)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", LOSSES + NARROW)
def test_loss(tr, shape, dt):
    n, k, v = shape
    dt = DTYPES[dt]
    h, w = rand(n, k, dtype=dt), rand(v, k, dtype=dt, std=2 * k ** -0.5, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(n + v)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    t[0], t[-1] = v - 1, 0
    if n > 4:
        t[2::5] = -100
    g = (0.5 + torch.rand(n, generator=gen, device="cuda")) * (1024.0 if dt == torch.float16 else 1.0) / n
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    _, wlse, wloss, valid, _ = loss_values(h, w, t)
    within(lse.sum(1), wlse, "lse")
    within(loss, wloss, "loss")
    assert not loss[~valid].any()
    dh, dw = tr.vocabulary_loss_backward(g, h, w, t, lse)
    for got, want, what in zip((dh, dw), loss_grads(g, h, w, t), ("dh", "dw")):
        within(got, want, what)
    assert not dh[~valid].any()
    for i in range(2):
        one = tr.vocabulary_loss_backward(g, h, w, t, lse, needs=(i == 0, i == 1))
        assert one[1 - i] is None and torch.equal(one[i], (dh, dw)[i])


def test_loss_every_row_ignored(tr):
    for dt in DTYPES.values():
        h, w = rand(20, 24, dtype=dt), rand(50, 24, dtype=dt)
        t = torch.full((20,), 7, device="cuda")
        loss, lse = tr.vocabulary_loss_forward(h, w, t, ignore_index=7)
        assert not loss.any() and torch.isfinite(lse).all()
        # what the upstream gradient holds for ignored rows does not matter
        dh, dw = tr.vocabulary_loss_backward(torch.full((20,), math.nan, device="cuda"), h, w, t, lse, ignore_index=7)
        assert not dh.any() and not dw.any() and torch.isfinite(dh).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(300, 72, 500), (5000, 40, 300), (200, 24, 19000), (4100, 16, 19001), (9000, 100, 130)])
def test_loss_ignored_rows_reach_nothing(tr, shape, dt):
    """Most rows are ignored and hold infinities and NaN: the gradients are those of the others alone."""
    n, k, v = shape
    dt = DTYPES[dt]
    h, w = rand(n, k, dtype=dt), rand(v, k, dtype=dt, std=k ** -0.5, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(n)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    out = torch.rand(n, generator=gen, device="cuda") < 0.7
    out[n // 3:n // 2] = True
    out[n - 1] = False
    t[out] = -100
    g = (0.5 + torch.rand(n, generator=gen, device="cuda")) / n * (1024.0 if dt == torch.float16 else 1.0)
    bad = h.clone()
    bad[out] = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda", dtype=dt)[
        torch.randint(0, 3, (int(out.sum()), 1), generator=gen, device="cuda")].expand(-1, k)
    loss, lse = tr.vocabulary_loss_forward(bad, w, t)
    assert not loss[out].any() and torch.isfinite(loss).all()
    dh, dw = tr.vocabulary_loss_backward(g, bad, w, t, lse)
    assert not dh[out].any() and torch.isfinite(dh).all() and torch.isfinite(dw).all()
    keep = ~out
    wdh, wdw = loss_grads(g[keep], h[keep], w, t[keep])
    within(dh[keep].contiguous(), wdh, "dh")
    within(dw, wdw, "dw")


def test_loss_target_out_of_range(tr):
    h, w = rand(6, 24, dtype=torch.bfloat16), rand(50, 24, dtype=torch.bfloat16)
    t = torch.tensor([0, 49, 50, -1, -100, 3], device="cuda")
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    assert torch.isnan(loss).tolist() == [False, False, True, True, False, False]
    dh, _ = tr.vocabulary_loss_backward(torch.ones(6, device="cuda"), h, w, t, lse)
    assert torch.isnan(dh).all(1).tolist() == [False, False, True, True, False, False]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_loss_very_negative_logits(tr, dt):
    """Every logit far below zero: what a tile computes past the vocabulary's end may overflow and has to stay out."""
    dt = DTYPES[dt]
    for v in (1, 5, 19001):
        h = torch.full((3, 16), 4.0, device="cuda", dtype=dt)
        w = torch.full((v, 16), -2.0, device="cuda", dtype=dt) + rand(v, 16, dtype=dt, std=0.01)
        t = torch.tensor([0, v - 1, v // 2], device="cuda")
        g = torch.ones(3, device="cuda")
        loss, lse = tr.vocabulary_loss_forward(h, w, t)
        within(loss, loss_values(h, w, t)[2], "loss")
        for got, want, what in zip(tr.vocabulary_loss_backward(g, h, w, t, lse), loss_grads(g, h, w, t), ("dh", "dw")):
            within(got, want, what)


def test_loss_large_logits(tr):
    """Logits of thousands, and vocabulary rows at the type's lowest value."""
    h = torch.tensor([[100.0, 1.0], [-100.0, 1.0]], device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(600, 2, device="cuda", dtype=torch.bfloat16)
    w[:, 0] = torch.linspace(-30, 30, 600).to(w.dtype)
    w[5:300, 1] = torch.finfo(torch.bfloat16).min  # a padded part of the vocabulary
    t = torch.tensor([599, 0], device="cuda")
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    l = h.double() @ w.double().T
    want = torch.logsumexp(l, 1)
    assert torch.allclose(lse.double().sum(1), want, rtol=1e-6)
    p = torch.softmax(l, 1)
    p[torch.arange(2), t] -= 1
    dh, dw = tr.vocabulary_loss_backward(torch.ones(2, device="cuda"), h, w, t, lse)
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all()
    wantw = p.T @ h.double()
    # p to 2^-9, its exponent of thousands to 3000 * 2^-22
    assert ((dw.double() - wantw).abs() <= 2.0 ** -7 * (p.abs().T @ h.double().abs()) + 1e-6).all()


def test_loss_pieces(tr):
    """Enough rows and columns that the backward pass takes the vocabulary in several pieces."""
    n, k, v = 16500, 40, 20011
    h, w = rand(n, k, dtype=torch.bfloat16), rand(v, k, dtype=torch.bfloat16, std=0.3)
    t = torch.randint(0, v, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    g = torch.full((n,), 1.0 / n, device="cuda")
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    dh, dw = tr.vocabulary_loss_backward(g, h, w, t, lse)
    _, wlse, wloss, _, _ = loss_values(h[::37], w, t[::37])
    within(loss[::37].contiguous(), wloss, "loss")
    wdh, _ = loss_grads(g[::37], h[::37], w, t[::37])
    within(dh[::37].contiguous(), wdh, "dh")
    wdw = torch.zeros(v, k, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(wdw)
    for i in range(0, n, 1500):
        hi = h[i:i + 1500].double()
        z = torch.softmax(hi @ w.double().T, 1)
        z[torch.arange(len(z)), t[i:i + 1500]] -= 1
        wdw += z.T @ hi / n
        mag += z.abs().T @ hi.abs() / n
    # Z rounded (2^-8), its exponential within 2^-17, n terms summed in 32 bits
    within(dw, V(wdw, mag * (2.0 ** -8 + 2.0 ** -17 + n * ACC)), "dw")


def test_loss_forward_pieces(tr):
    """So many rows over so large a vocabulary that the forward pass takes the rows in several pieces."""
    n, k, v = 9000, 16, 2100003
    h, w = rand(n, k, dtype=torch.bfloat16), rand(v, k, dtype=torch.bfloat16, std=0.25)
    t = torch.randint(0, v, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    loss, lse = tr.vocabulary_loss_forward(h, w, t)
    rows = torch.tensor([0, 1, 4095, 4096, 4097, 8191, 8192, 8999], device="cuda")
    _, wlse, wloss, _, _ = loss_values(h[rows], w, t[rows])
    within(lse[rows].sum(1), wlse, "lse")
    within(loss[rows], wloss, "loss")
    one, _ = tr.vocabulary_loss_forward(h[:100], w, t[:100])
    assert torch.equal(one, loss[:100])


# ------------------------------------------------------------------ gradients against differences
def test_gated_differences(tr):
    """h is quadratic in x for the identity gate, so the central difference
    is exact up to the rounding of h; for silu the third derivative bounds it."""
    dt = torch.float16
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randint(-8, 9, (24, 40), generator=gen, device="cuda").to(dt) / 8
    wg = torch.randint(-8, 9, (56, 40), generator=gen, device="cuda").to(dt) / 32
    wu = torch.randint(-8, 9, (56, 40), generator=gen, device="cuda").to(dt) / 32
    dh = torch.randint(-4, 5, (24, 56), generator=gen, device="cuda").to(dt) / 4
    for name, step in (("identity", 0.5), ("silu", 0.125)):
        grads = tr.gated_backward(dh, x, wg, wu, name)
        bounds = [rnd(v, dt).e for v in gated_grads(dh, x, wg, wu, name)]
        for which, at in ((0, (3, 7)), (0, (23, 39)), (1, (0, 0)), (1, (55, 20)), (2, (17, 11))):
            def h(sign):
                a = [x.clone(), wg.clone(), wu.clone()]
                a[which][at] += sign * step
                return tr.gated_forward(*a, name).double()
            hp, hm = h(1), h(-1)
            diff = float((dh.double() * (hp - hm)).sum() / (2 * step))
            tol = float((dh.double().abs() * (hp.abs() + hm.abs())).sum()) * 1.01 * 2.0 ** -11 / (2 * step)
            if name == "silu":  # |d^3 h| <= |silu'''| s^3 |u| + 3 |silu''| s^2 s', s the slopes: weights or x, at most 1
                u = (x.double() @ wu.double().T).abs() + 0.25
                s = 0.25 if which == 0 else 1.0
                rows = dh.double().abs() * (0.35 * s ** 3 * u + 3 * 0.5 * s ** 3)
                tol += step ** 2 / 6 * float(rows.sum() if which else rows[at[0]].sum())
            assert abs(diff - float(grads[which][at])) <= tol + float(bounds[which][at]), (name, which, at)


def test_loss_differences(tr):
    dt = torch.float16
    gen = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randint(-8, 9, (30, 16), generator=gen, device="cuda").to(dt) / 8
    w = torch.randint(-8, 9, (70, 16), generator=gen, device="cuda").to(dt) / 16
    t = torch.randint(0, 70, (30,), generator=gen, device="cuda")
    t[4] = -100
    g = torch.ones(30, device="cuda")
    _, lse = tr.vocabulary_loss_forward(h, w, t)
    grads = tr.vocabulary_loss_backward(g, h, w, t, lse)
    bounds = [rnd(v, dt).e for v in loss_grads(g, h, w, t)]
    step = 2.0 ** -5
    for which, at in ((0, (0, 0)), (0, (29, 15)), (0, (4, 3)), (1, (0, 0)), (1, (69, 15)), (1, (int(t[1]), 5))):
        def total(sign):
            a = [h.clone(), w.clone()]
            a[which][at] += sign * step
            return float(tr.vocabulary_loss_forward(*a, t)[0].double().sum())
        diff = (total(1) - total(-1)) / (2 * step)
        # the third derivative of lse is a third central moment: at most R^3 / (6 sqrt 3), R the range of the slopes
        # (1 for h and w both); a row each for w
        tol = step ** 2 / 6 * 0.0963 * (1 if which == 0 else 30) * 2 ** 3
        tol += 30 * 2 * 6.0 * 2.0 ** -20 / (2 * step)  # the losses themselves
        assert abs(diff - float(grads[which][at])) <= tol + float(bounds[which][at]), (which, at)


# ------------------------------------------------------------------ as a user has them
@pytest.mark.parametrize("keep", [False, True])
def test_autograd(tr, keep):
    dt = torch.bfloat16
    x, wg, wu, _ = block((50, 40, 24), dt)
    w = rand(90, 24, dtype=dt, std=0.4, seed=9)
    t = torch.randint(0, 90, (5, 10), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    t[0, 0] = -100
    leaves = [v.clone().requires_grad_() for v in (x.view(5, 10, 40), wg, wu, w)]
    h = tr.gated_feed_forward(*leaves[:3], "silu", checkpoint=keep)
    loss = tr.vocabulary_cross_entropy(h, leaves[3], t)
    loss.backward()
    n = 49
    hh = tr.gated_forward(x, wg, wu)
    rows, lse = tr.vocabulary_loss_forward(hh, w, t.view(-1))
    assert torch.allclose(loss.detach(), rows.sum() / n)
    dh, dw = tr.vocabulary_loss_backward(torch.full((50,), 1.0 / n, device="cuda"), hh, w, t.view(-1), lse)
    kept = tr.pack_checkpoint(x) if keep else x
    want = (*tr.gated_backward(dh, kept, wg, wu), dw)
    for leaf, v in zip(leaves, want):
        assert torch.equal(leaf.grad.reshape(v.shape), v)
    assert torch.equal(tr.vocabulary_cross_entropy(hh, w, t.view(-1), reduction="none"), rows)
    assert torch.equal(tr.vocabulary_cross_entropy(hh, w, t.view(-1), reduction="sum"), rows.sum())


def test_autograd_of_a_frozen_part(tr):
    x, wg, wu, _ = block((50, 40, 24), torch.float16)
    wg = wg.clone().requires_grad_()
    h = tr.gated_feed_forward(x, wg, wu, "relu")
    h.float().sum().backward()
    want = tr.gated_backward(torch.ones_like(h), x, wg.detach(), wu, "relu")
    assert torch.equal(wg.grad, want[1]) and wu.grad is None
    # a weight used twice gets the sum of both gradients
    wg.grad = None
    (tr.gated_feed_forward(x, wg, wu, "relu").float().sum() + tr.gated_feed_forward(x, wg, wu, "relu").float().sum()).backward()
    assert torch.equal(wg.grad, want[1] + want[1])


def test_same_bits_and_other_streams(tr):
    x, wg, wu, dh = block((700, 136, 520), torch.bfloat16)
    w = rand(3000, 136, dtype=torch.bfloat16, std=0.2, seed=4)
    t = torch.randint(0, 3000, (700,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    g = torch.rand(700, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))

    def every():
        c = tr.pack_checkpoint(x)
        loss, lse = tr.vocabulary_loss_forward(x, w, t)
        return [tr.gated_forward(x, wg, wu), *tr.gated_backward(dh, c, wg, wu), loss, lse,
                *tr.vocabulary_loss_backward(g, x, w, t, lse)]

    ref = every()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(every())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, ref))


def test_in_a_graph(tr):
    x, wg, wu, dh = block((300, 136, 200), torch.bfloat16)
    w = rand(3000, 136, dtype=torch.bfloat16, std=0.2, seed=4)
    t = torch.randint(0, 3000, (300,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))

    def every():
        loss, lse = tr.vocabulary_loss_forward(x, w, t)
        return [tr.gated_forward(x, wg, wu), *tr.gated_backward(dh, x, wg, wu), loss,
                *tr.vocabulary_loss_backward(loss, x, w, t, lse)]

    every()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = every()
    x.copy_(rand(300, 136, dtype=torch.bfloat16, seed=77))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, every()))


# ------------------------------------------------------------------ refusals
def test_refusals(tr):
    x, wg, wu, dh = block((10, 40, 24), torch.bfloat16)
    t = torch.zeros(10, dtype=torch.int64, device="cuda")
    bad = [
        lambda: tr.gated_forward(x.float(), wg, wu),
        lambda: tr.gated_forward(x.cpu(), wg, wu),
        lambda: tr.gated_forward(x, wg.half(), wu),
        lambda: tr.gated_forward(x, wg.cpu(), wu),
        lambda: tr.gated_forward(x, wg[:, :39], wu),
        lambda: tr.gated_forward(x, wg[:23], wu),
        lambda: tr.gated_forward(x, wg[:0], wu[:0]),
        lambda: tr.gated_forward(x, wg.view(2, 12, 40), wu),
        lambda: tr.gated_forward(x, wg, wu, "tanh"),
        lambda: tr.gated_forward(x[:, :0], wg[:, :0], wu[:, :0]),
        lambda: tr.gated_forward(None, wg, wu),
        lambda: tr.gated_backward(dh[:9], x, wg, wu),
        lambda: tr.gated_backward(dh[:, :23], x, wg, wu),
        lambda: tr.gated_backward(dh.half(), x, wg, wu),
        lambda: tr.gated_backward(dh.half(), tr.pack_checkpoint(x), wg.half(), wu.half()),
        lambda: tr.gated_backward(dh, tr.pack_checkpoint(x)._replace(shape=(10, 72)), wg, wu),
        lambda: tr.gated_backward(dh, tr.pack_checkpoint(x)._replace(q=torch.zeros(3, device="cuda")), wg, wu),
        lambda: tr.pack_checkpoint(x.double()),
        lambda: tr.unpack_checkpoint(x),
        lambda: tr.unpack_checkpoint(tr.pack_checkpoint(x)._replace(shape=(11, 40))),
        lambda: tr.vocabulary_loss_forward(x, wg[:, :8], t),
        lambda: tr.vocabulary_loss_forward(x, wg[:0], t),
        lambda: tr.vocabulary_loss_forward(x, wg, t[:9]),
        lambda: tr.vocabulary_loss_forward(x, wg, t.float()),
        lambda: tr.vocabulary_loss_forward(x, wg, t.cpu()),
        lambda: tr.vocabulary_loss_backward(torch.zeros(9, device="cuda"), x, wg, t, torch.zeros(10, 2, device="cuda")),
        lambda: tr.vocabulary_loss_backward(torch.zeros(10, device="cuda"), x, wg, t,
                                            torch.zeros(10, 2, device="cuda", dtype=torch.float64)),
        lambda: tr.vocabulary_loss_backward(torch.zeros(10, device="cuda"), x, wg, t, torch.zeros(10, device="cuda")),
        lambda: tr.vocabulary_cross_entropy(x, wg, t, reduction="median"),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()


def test_refusals_of_the_c_entries(tr):
    """Status codes and messages at the C boundary; nothing is launched."""
    import ctypes

    from helrm_b200 import _capi
    lib = _capi.load()
    x, wg, wu, _ = block((10, 40, 24), torch.bfloat16)
    h = torch.empty(10, 24, dtype=torch.bfloat16, device="cuda")
    need = ctypes.c_size_t(0)

    def forward(device=0, dtype=1, act=2, tokens=10, inner=40, width=24, xp=x.data_ptr(), ldx=40, ws=None,
                size=ctypes.byref(need)):
        return lib.helrm_GatedForward(device, dtype, act, tokens, inner, width, xp, ldx, wg.data_ptr(), 40,
                                      wu.data_ptr(), 40, h.data_ptr(), ws, size, None)

    assert forward() == 0
    ws = torch.empty(need.value + 512, dtype=torch.uint8, device="cuda")
    ok = ctypes.c_size_t(need.value)
    for kw in (dict(dtype=2), dict(act=4), dict(act=-1), dict(tokens=-1), dict(inner=0), dict(width=0), dict(xp=None),
               dict(xp=x.data_ptr() + 1), dict(ldx=39), dict(size=None), dict(inner=2 ** 31),
               dict(ws=ws.data_ptr() + 8, size=ctypes.byref(ok)),
               dict(ws=ws.data_ptr(), device=99, size=ctypes.byref(ok)),
               dict(ws=ws.data_ptr(), device=-1, size=ctypes.byref(ok))):
        assert forward(**kw) == -1, kw
        with pytest.raises(ValueError):
            _capi.check(-1)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ long tensors
def test_offsets_past_32_bits(tr):
    """Results and inputs of more than 2^31 elements: their last rows are right."""
    dt = torch.bfloat16
    t, k, f = 140001, 16, 16384  # h: 2.3e9 elements
    x, wg, wu = rand(t, k, dtype=dt), rand(f, k, dtype=dt, std=0.25, seed=1), rand(f, k, dtype=dt, std=0.25, seed=2)
    h = tr.gated_forward(x, wg, wu)
    assert h.numel() > 2 ** 31
    rows = torch.tensor([0, 131071, 131072, 139999, 140000], device="cuda")
    within(h[rows], gated(x[rows], wg, wu, "silu"), "h")
    c = tr.pack_checkpoint(h)
    back = tr.unpack_checkpoint(c)
    assert torch.equal(back[rows], tr.unpack_checkpoint(tr.pack_checkpoint(h[rows])))
    # dh as long: its gradients over the last rows alone
    dx, _, _ = tr.gated_backward(h, x, wg, wu, needs=(True, False, False))
    within(dx[rows], gated_grads(h[rows], x[rows], wg, wu, "silu")[0], "dx")
    del h, c, back, dx
    v, k, n = 1060000, 2048, 130  # w: 2.2e9 elements
    w = torch.empty(v, k, dtype=dt, device="cuda")
    for i in range(0, v, 106000):
        w[i:i + 106000] = rand(106000, k, dtype=dt, std=k ** -0.5, seed=i)
    assert w.numel() > 2 ** 31
    x = rand(n, k, dtype=dt)
    t = torch.full((n,), v - 1, device="cuda")
    t[::2] = 0
    loss, lse = tr.vocabulary_loss_forward(x, w, t)
    ends = torch.stack([w[0], w[-1]])
    at = (x.double() @ ends.double().T).gather(1, (t > 0).long()[:, None])[:, 0]
    top = torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(0, v, 106000):
        top = torch.logaddexp(top, torch.logsumexp(x.double() @ w[i:i + 106000].double().T, 1))
    assert ((loss.double() - (top - at)).abs() < 1e-4).all()
    dh, dw = tr.vocabulary_loss_backward(torch.ones(n, device="cuda"), x, w, t, lse)
    z = torch.exp(x.double() @ ends.double().T - top[:, None])
    z[:, 0] -= (t == 0).double()
    z[:, 1] -= (t > 0).double()
    want = z.T @ x.double()
    mag = z.abs().T @ x.double().abs()
    # z to 2^-8 and 1e-4 of its exponential, 130 terms in 32 bits, the result to 2^-8
    assert ((dw[[0, -1]].double() - want).abs() <= mag * (2.0 ** -8 + 1.5e-4) + 2.0 ** -8 * want.abs()).all()
    assert torch.isfinite(dh).all()
