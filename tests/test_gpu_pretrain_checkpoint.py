"""The example keeps an 8-bit copy of the block's input where it is asked to."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_training import give_memory_back  # noqa: E402,F401


@pytest.mark.parametrize("checkpoint", [False, True])
def test_input_kept_in_eight_bits_only_if_asked(monkeypatch, checkpoint):
    from helrm_b200 import pretrain, training
    packed = []
    pack = training.pack_checkpoint
    monkeypatch.setattr(training, "pack_checkpoint", lambda x: packed.append(tuple(x.shape)) or pack(x))
    weights, losses = pretrain.train(steps=40, rows=1024, width=32, vocab=300, **({"checkpoint": True} if checkpoint else {}))
    assert packed == ([(1024, 13)] * 40 if checkpoint else [])
    assert all(math.isfinite(v) for v in losses) and losses[-1] < losses[0] - 0.3
    assert all(torch.isfinite(w).all() for w in weights.values())
