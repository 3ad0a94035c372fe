"""The training operators' calls at their edges, without a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from helrm_b200 import _capi, build
    build.build()
    return _capi.load()


def test_an_empty_gradient_needs_no_address(lib):
    """With no tokens the input's gradient has no elements, so its address may be NULL though it is asked for."""
    n = ctypes.c_size_t(0)
    p = 4096  # an address: the size query reads nothing

    def gated(tokens, dx, dwg):
        return lib.helrm_GatedBackward(0, 1, 2, tokens, 40, 24, p, 24, p, 40, None, None, p, 40, p, 40, dx, dwg, None, None,
                                       ctypes.byref(n), None)

    def loss(tokens, vocab, dh, dw):
        return lib.helrm_VocabularyLossBackward(0, 1, tokens, 40, vocab, p, p, 40, p, 40, p, p, -100, dh, dw, None,
                                                ctypes.byref(n), None)

    assert gated(0, None, None) == 0 and gated(0, None, p) == 0
    assert gated(3, None, None) == -1 and gated(3, p, None) == 0
    for vocab in (300, 40000):
        assert loss(0, vocab, None, None) == 0 and loss(3, vocab, None, None) == -1


def test_what_is_no_checkpoint_is_refused():
    """ValueError, whichever part is not what pack_checkpoint returns."""
    from helrm_b200 import training as tr
    q, e = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8)
    good = dict(q=q, e=e, shape=(4, 8), dtype=torch.bfloat16)
    for part in (dict(q=None), dict(q=[1, 2]), dict(q=q.numpy()), dict(e=None), dict(e=3), dict(shape=None), dict(shape=8),
                 dict(shape=()), dict(shape=("a", 8)), dict(shape=[4, 8]), dict(dtype=None), dict(dtype=[]),
                 dict(dtype="bf16"), dict(dtype=torch.float32)):
        for _ in range(2):
            with pytest.raises(ValueError):
                tr.unpack_checkpoint(tr.Checkpoint(**{**good, **part}))
    assert None not in tr._plans


def test_an_activation_that_is_no_name_is_refused():
    from helrm_b200 import training as tr
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    for bad in ([], {}, None, 2, "tanh"):
        with pytest.raises(ValueError):
            tr.gated_forward(x, x, x, bad)
        with pytest.raises(ValueError):
            tr.gated_backward(x, x, x, x, bad)


def test_nothing_is_kept_where_no_gradient_is_recorded(monkeypatch):
    """Stand-ins for the passes, since they take no tensors of the CPU."""
    from helrm_b200 import training as tr
    packed = []

    def pack(x):
        packed.append(x.shape)
        return tr.Checkpoint(x.clone(), x.clone(), tuple(x.shape), x.dtype)
    monkeypatch.setattr(tr, "pack_checkpoint", pack)
    monkeypatch.setattr(tr, "gated_forward", lambda x, wg, wu, act: (x @ wg.T) * (x @ wu.T))
    x, w = torch.ones(4, 8), torch.ones(6, 8)
    assert not tr.gated_feed_forward(x, w, w, checkpoint=True).requires_grad and not packed
    for leaf in range(3):
        args = [t.clone().requires_grad_(i == leaf) for i, t in enumerate((x, w, w))]
        with torch.no_grad():
            assert not tr.gated_feed_forward(*args, checkpoint=True).requires_grad and not packed
        with torch.inference_mode():
            assert not tr.gated_feed_forward(*args, checkpoint=True).requires_grad and not packed
        assert tr.gated_feed_forward(*args, checkpoint=True).requires_grad and len(packed) == 1
        packed.clear()


def test_an_ignore_index_that_is_no_whole_number_is_refused():
    """A half would leave rows out of the loss and not out of its mean."""
    from helrm_b200 import training as tr
    x, t = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    for bad in (-100.5, 7.0, None, "7", 2 ** 63, -2 ** 63 - 1):
        for call in (lambda: tr.vocabulary_loss_forward(x, x, t, bad), lambda: tr.vocabulary_cross_entropy(x, x, t, bad),
                     lambda: tr.vocabulary_loss_backward(x, x, x, t, x, bad)):
            with pytest.raises(ValueError, match="ignore_index"):
                call()


def test_each_thread_reads_its_own_failure(lib):
    """Two threads fail in turn, each then reads; a third one that has not failed finds the process's last."""
    import threading
    n = ctypes.c_size_t(0)

    def fail(**kw):
        a = dict(dtype=1, inner=40, ldx=40)
        a.update(kw)
        assert lib.helrm_GatedForward(0, a["dtype"], 2, 3, a["inner"], 24, 4096, a["ldx"], 4096, 40, 4096, 40, 4096, None,
                                      ctypes.byref(n), None) == -1

    turn = threading.Barrier(2)
    got = {}

    def run(name, first, **kw):
        if not first:
            turn.wait()
        fail(**kw)
        if first:
            turn.wait()
        turn.wait()  # both have failed
        got[name] = lib.helrm_LastError()
    threads = [threading.Thread(target=run, args=("dtype", True), kwargs=dict(dtype=7)),
               threading.Thread(target=run, args=("pitch", False), kwargs=dict(ldx=3))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert b"dtype" in got["dtype"] and b"pitch" in got["pitch"]
    other = threading.Thread(target=lambda: got.update(other=lib.helrm_LastError()))
    other.start()
    other.join()
    assert b"pitch" in got["other"]
    fail(inner=0)
    assert b"sizes" in lib.helrm_LastError()


@pytest.mark.skipif(torch.cuda.is_available(), reason="what a host without a GPU answers")
def test_no_device_is_an_error_code(lib):
    assert lib.helrm_TrainingSynchronize(0, None) < 0 and lib.helrm_LastError()
    assert lib.helrm_TrainingPostFailure(0, 4) < 0
    assert lib.helrm_TrainingPostFailure(0, 0) == -1
