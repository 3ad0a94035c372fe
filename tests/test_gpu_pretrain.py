"""A gated model trained in the clear and answered on ciphertexts."""
import gc
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def give_memory_back():
    """The tests after these find torch's allocator as if these had not run."""
    yield
    gc.collect()
    torch.cuda.empty_cache()


def test_trained_model_runs_encrypted():
    from helrm_b200 import pretrain
    r = pretrain.main(["--steps", "120", "--rows", "2048", "--vocab", "500", "--width", "48", "--queries", "3"])
    losses = r["losses"]
    assert len(losses) == 120 and all(math.isfinite(v) for v in losses)
    # it starts near a guess (the logarithm of 500) and learns
    assert abs(losses[0] - math.log(500)) < 1.5 and losses[-1] < losses[0] - 1.0
    w = {n: v.double().cpu().numpy() for n, v in r["weights"].items()}
    x = r["x"].double().cpu().numpy()
    want = ((x @ w["w_gate"].T) * (x @ w["w_up"].T)) @ w["w_out"].T
    # the ciphertexts against 64 bits; the clear model against them by the rounding of h to bfloat16
    assert np.abs(r["logits"] - want).max() < 1e-3 * max(1.0, np.abs(want).max())
    h = np.abs((x @ w["w_gate"].T) * (x @ w["w_up"].T))
    assert (np.abs(r["clear"] - want) <= 2.0 ** -8 * 1.01 * (h @ np.abs(w["w_out"]).T) + 1e-6).all()
