"""The training operators without a GPU: what they refuse before any launch,
the C entries' argument checks and workspace sizes, the example's data."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def capi():
    from helrm_b200 import _capi, build
    build.build()
    return _capi, _capi.load()


def test_tensors_of_the_cpu_are_refused(capi):
    from helrm_b200 import training as tr
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    c = tr.Checkpoint(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8), (4, 8), x.dtype)
    dh = torch.zeros(4, 6, dtype=torch.bfloat16)
    for call in (lambda: tr.gated_forward(x, w, w), lambda: tr.gated_backward(dh, x, w, w),
                 lambda: tr.gated_backward(dh, c, w, w), lambda: tr.pack_checkpoint(x),
                 lambda: tr.unpack_checkpoint(c), lambda: tr.vocabulary_loss_forward(x, w, t),
                 lambda: tr.gated_feed_forward(x, w, w), lambda: tr.vocabulary_cross_entropy(x, w, t)):
        for _ in range(2):  # the second time as the first
            with pytest.raises(ValueError):
                call()


def test_what_is_no_tensor_is_refused(capi):
    from helrm_b200 import training as tr
    for bad in (None, 3.0, [[1.0]], np.zeros((4, 8))):
        with pytest.raises(ValueError):
            tr.gated_forward(bad, bad, bad)
        with pytest.raises(ValueError):
            tr.pack_checkpoint(bad)
        with pytest.raises(ValueError):
            tr.unpack_checkpoint(bad)
        with pytest.raises(ValueError):
            tr.vocabulary_loss_forward(bad, bad, bad)


def test_c_entries_check_before_they_launch(capi):
    mod, lib = capi
    n = ctypes.c_size_t(0)
    p = 4096  # an address: the size query reads nothing

    def loss(dtype=1, tokens=5, inner=16, vocab=100, h=p, ldh=16, w=p, ldw=16, targets=p, out=p, ws=None, size=n):
        return lib.helrm_VocabularyLossForward(0, dtype, tokens, inner, vocab, h, ldh, w, ldw, targets, -100, out, out, ws,
                                               None if size is None else ctypes.byref(size), None)

    assert loss() == 0 and n.value > 0
    for kw in (dict(dtype=-1), dict(tokens=-1), dict(inner=0), dict(vocab=0), dict(h=None), dict(w=None), dict(ldh=15),
               dict(ldw=15), dict(targets=None), dict(out=None), dict(out=p + 4), dict(h=p + 1), dict(size=None),
               dict(vocab=1 << 31), dict(ws=p + 8), dict(ws=p, size=ctypes.c_size_t(1))):
        assert loss(**kw) == -1, kw
        assert lib.helrm_LastError()
    assert loss(tokens=0, h=None, targets=None, out=None) == 0
    for call in (lambda: lib.helrm_PackCheckpoint(0, 1, 4, 0, p, 8, p, p, None),
                 lambda: lib.helrm_PackCheckpoint(0, 1, 4, 8, p, 7, p, p, None),
                 lambda: lib.helrm_PackCheckpoint(0, 1, 4, 8, p, 8, p + 8, p, None),
                 lambda: lib.helrm_PackCheckpoint(0, 1, 4, 8, p, 8, p, None, None),
                 lambda: lib.helrm_UnpackCheckpoint(0, 1, 4, 8, p, p, None, None),
                 lambda: lib.helrm_UnpackCheckpoint(0, 3, 4, 8, p, p, p, None)):
        assert call() == -1
    assert lib.helrm_PackCheckpoint(0, 1, 0, 8, p, 8, None, None, None) == 0


def test_workspaces_grow_with_what_needs_copies(capi):
    _, lib = capi

    def size(ldx, x=4096):
        n = ctypes.c_size_t(0)
        assert lib.helrm_GatedForward(0, 1, 2, 100, 13, 24, x, ldx, 4096, 16, 4096, 16, 4096, None, ctypes.byref(n),
                                      None) == 0
        return n.value

    assert size(16) == 0                # rows on 16-byte boundaries are read as they are
    assert size(13) >= 100 * 16 * 2     # others are copied
    assert size(16, 4098) == size(13)


def test_example_data():
    from helrm_b200 import pretrain
    x, y = pretrain.make_data(200, 50, seed=1)
    assert x.shape == (200, 13) and y.shape == (200,) and y.min() >= 0 and y.max() < 50
    x2, y2 = pretrain.make_data(200, 50, seed=1)
    assert np.array_equal(x, x2) and np.array_equal(y, y2)
    assert not np.array_equal(x, pretrain.make_data(200, 50, seed=2)[0])
    for bad in (["--vocab", "0"], ["--vocab", "4096"], ["--steps", "0"]):
        with pytest.raises(SystemExit):
            pretrain.main(bad)
