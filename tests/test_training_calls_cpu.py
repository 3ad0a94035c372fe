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
