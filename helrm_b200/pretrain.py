"""Train a small gated model in the clear, then evaluate it on ciphertexts.

    python -m helrm_b200.pretrain [--steps 200] [--rows 4096] [--width 64] [--vocab 1000] [--checkpoint]

The model predicts one categorical field from the 13 dense features: a gated
feed-forward block with the identity activation, then a row of weights for
every category, trained with the softmax cross entropy over the vocabulary
(:mod:`helrm_b200.training`; with --checkpoint the block keeps its input in 8
bits for the backward pass, which pays for more features than these).  What
was trained needs nothing a ciphertext cannot do: two linear transforms, one
ciphertext product and a third transform, three levels.  The trained weights
go to the backend's linear layers and a few queries are answered encrypted and
compared with the clear model's logits.

Data are synthetic: log1p(lognormal) features, categories drawn from a
random model of the same form.
"""
from __future__ import annotations

import argparse

import numpy as np

from .helrm import DENSE, dense_inputs
from .library import B200Library
from .mlp import LinearLayer
from .params import CKKSConfig

# three levels for the model above a 40-bit base, 2048 slots
CKKS = CKKSConfig(logn=12, logq=[40] + [36] * 5, logp=[60, 60], logscale=36, h=64)


def make_data(rows: int, vocab: int, seed: int):
    """(features [rows, 13], categories [rows])"""
    x = dense_inputs(rows, seed)
    rng = np.random.default_rng(1234)  # one teacher for every split
    a, b = rng.normal(0, DENSE ** -0.5, (2, DENSE, 32))
    w = rng.normal(0, 1.5, (32, vocab))
    logits = ((x @ a) * (x @ b)) @ w
    gumbel = -np.log(-np.log(np.random.default_rng(seed + 1).uniform(1e-12, 1, logits.shape)))
    return x, (logits + gumbel).argmax(1)


def train(steps: int = 200, rows: int = 4096, width: int = 64, vocab: int = 1000, seed: int = 0, report=None,
          checkpoint: bool = False):
    """The trained weights (w_gate, w_up [width, 13], w_out [vocab, width],
    bfloat16) and the loss of every step."""
    import torch

    from . import training

    gen = torch.Generator().manual_seed(seed)
    shapes = {"w_gate": (width, DENSE), "w_up": (width, DENSE), "w_out": (vocab, width)}
    master = [torch.nn.Parameter((torch.randn(s, generator=gen) * s[1] ** -0.5).cuda()) for s in shapes.values()]
    opt = torch.optim.Adam(master, lr=1e-2)
    x, y = make_data(rows, vocab, seed)
    x = torch.tensor(x, device="cuda").to(torch.bfloat16)
    y = torch.tensor(y, device="cuda")
    losses = []
    for i in range(steps):
        w_gate, w_up, w_out = (p.to(torch.bfloat16) for p in master)  # gradients come back to the 32-bit weights
        h = training.gated_feed_forward(x, w_gate, w_up, "identity", checkpoint=checkpoint)
        loss = training.vocabulary_cross_entropy(h, w_out, y)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if report and (i % 20 == 0 or i + 1 == steps):
            report(f"step {i}: loss {float(losses[-1]):.4f}")
    weights = {n: p.detach().to(torch.bfloat16) for n, p in zip(shapes, master)}
    return weights, [float(v) for v in losses]


class EncryptedGated:
    """The trained model on ciphertexts of a B200Library scheme: three levels."""

    def __init__(self, lib, weights, level: int):
        self.lib, self.level = lib, level
        w = {n: v.float().cpu().numpy() for n, v in weights.items()}
        self.gate = LinearLayer(lib, w["w_gate"], None, level, narrow=False)
        self.up = LinearLayer(lib, w["w_up"], None, level, narrow=False)
        self.out = LinearLayer(lib, w["w_out"], None, level - 2, narrow=False)

    def forward(self, cts) -> list[int]:
        lib = self.lib
        g, u = self.gate.forward(cts), self.up.forward(cts)
        h = lib.MulRelinCiphertextBatchNew(g, u)
        lib.RescaleBatch(h)
        y = self.out.forward(h)
        for c in g + u + h:
            lib.DeleteCiphertext(c)
        return y

    def close(self):
        for layer in (self.gate, self.up, self.out):
            layer.close()


def answer_encrypted(weights, x, seed: int = 7):
    """Logits [len(x), vocab] of the queries x [n, 13], decrypted after the
    encrypted forward."""
    vocab = weights["w_out"].shape[0]
    lib = B200Library(dnum=3, seed=seed, device=0)
    lib.setup_bindings(CKKS)
    try:
        lib.GenerateSecretKey()
        lib.GenerateRelinearizationKey()
        level = lib.scheme_info()["max_level"]
        model = EncryptedGated(lib, weights, level)
        pts = lib.EncodeBatch(np.asarray(x, dtype=np.float64), level, float(1 << CKKS.logscale))
        out = model.forward([lib.Encrypt(p) for p in pts])
        logits = np.stack([np.array(lib.Decode(lib.Decrypt(c)))[:vocab] for c in out])
        model.close()
        return logits
    finally:
        lib.DeleteScheme()


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--rows", type=int, default=4096)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--vocab", type=int, default=1000)
    ap.add_argument("--queries", type=int, default=4)
    ap.add_argument("--checkpoint", action="store_true",
                    help="keep the block's input in 8 bits for the backward pass (a row of 13 features takes 33 bytes "
                         "then instead of 26; of 17 or more, less)")
    a = ap.parse_args(argv)
    slots = 1 << (CKKS.logn - 1)
    if not 1 <= a.vocab <= slots or not 1 <= a.width <= slots:
        ap.error(f"--vocab and --width are 1 to {slots}, the ciphertext's slots")
    if a.steps < 1 or a.rows < 1 or a.queries < 1:
        ap.error("--steps, --rows and --queries are at least 1")
    import torch

    from . import training

    weights, losses = train(a.steps, a.rows, a.width, a.vocab, report=print, checkpoint=a.checkpoint)
    x = torch.tensor(make_data(a.queries, a.vocab, seed=99)[0], device="cuda").to(torch.bfloat16)
    h = training.gated_forward(x, weights["w_gate"], weights["w_up"], "identity")
    clear = (h.double() @ weights["w_out"].double().T).cpu().numpy()
    logits = answer_encrypted(weights, x.double().cpu().numpy())
    err = float(np.abs(logits - clear).max())
    same = int((logits.argmax(1) == clear.argmax(1)).sum())
    print(f"encrypted: {a.queries} queries, logits within {err:.3g} of the clear model's "
          f"(largest {np.abs(clear).max():.3g}), {same} of {a.queries} answers the same")
    return {"losses": losses, "logits": logits, "clear": clear, "weights": weights, "x": x}


if __name__ == "__main__":
    main()
