"""Cases that measure the training operators of ``helrm_b200.training``.

The encrypted model evaluates weights that were trained in the clear.  The
operators measured here are the ones that training spends its time in:

* ``gated``: the gated feed-forward block  H = act(X Wg^T) * (X Wu^T),
  forward, and ``gated_backward``: dX, dWg, dWu from dH, X, Wg, Wu;
* ``checkpoint``: an activation written in 8 bits (groups of 32 consecutive
  features share a power-of-two scale) and read back, and ``checkpointed``:
  a step of the gated block whose backward pass starts from that 8-bit copy;
* ``loss``: softmax cross entropy of H W^T over a vocabulary of V rows, a
  loss for each row, and ``loss_step``: with dH and dW.

Where ``own`` is false the operators run in plain torch arithmetic in 32
bits, rounded once at the end; where it is true, as a user calls the
framework.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP = 32       # features that share a scale in an 8-bit checkpoint
IGNORE = -100    # target of a row that takes no part in the loss
LARGEST = 2.7e13  # flops of the largest listed case; no drawn case has more


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a serving batch of 64 queries through the top model's first width: one short call, latency counts
        {"name": "gated 64 rows", "op": "gated", "tokens": 64, "inner": 432, "width": 512, "act": "silu",
         "dtype": "bf16"},
        # the 13 dense features, a row pitch that no vector load fits, the activation a ciphertext product evaluates
        {"name": "gated 13 features", "op": "gated", "tokens": 4096, "inner": 13, "width": 512, "act": "identity",
         "dtype": "fp16"},
        # a long training batch through a wide block
        {"name": "gated wide", "op": "gated", "tokens": 16384, "inner": 4096, "width": 12288, "act": "silu",
         "dtype": "bf16"},
        # an ordinary training batch's backward pass
        {"name": "gated backward", "op": "gated_backward", "tokens": 4096, "inner": 1024, "width": 4096,
         "act": "gelu", "dtype": "bf16"},
        # the backward pass of a wide block
        {"name": "gated backward wide", "op": "gated_backward", "tokens": 8192, "inner": 4096, "width": 12288,
         "act": "silu", "dtype": "bf16"},
        # a step from an 8-bit copy, ragged in every size
        {"name": "checkpointed ragged", "op": "checkpointed", "tokens": 2047, "inner": 1001, "width": 1500,
         "act": "relu", "dtype": "fp16"},
        # a small activation kept in 8 bits: one short call each way
        {"name": "checkpoint small", "op": "checkpoint", "tokens": 256, "inner": 512, "dtype": "bf16"},
        # the activation of a long batch kept in 8 bits
        {"name": "checkpoint long", "op": "checkpoint", "tokens": 32768, "inner": 4096, "dtype": "bf16"},
        # a validation pass over one categorical field: the loss alone
        {"name": "loss small field", "op": "loss", "tokens": 64, "inner": 64, "vocab": 1000, "ignored": 0.0,
         "dtype": "bf16"},
        # a field of a million categories at the embedding tables' width
        {"name": "loss step wide field", "op": "loss_step", "tokens": 1024, "inner": 16, "vocab": 1000003,
         "ignored": 0.05, "dtype": "bf16"},
        # ragged in every size, a third of the rows without a target, scaled for the type's range
        {"name": "loss step ragged", "op": "loss_step", "tokens": 777, "inner": 432, "vocab": 32001,
         "ignored": 0.33, "dtype": "fp16"},
        # a long batch over a large vocabulary: the largest
        {"name": "loss step large", "op": "loss_step", "tokens": 8192, "inner": 4096, "vocab": 131072,
         "ignored": 0.05, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm; one of three is a multiple of 64 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.34 and v > 64:
        v = v // 64 * 64
    v = min(hi, max(lo, v))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["gated", "gated_backward", "checkpointed", "checkpoint", "loss", "loss_step"])
    dtype = rng.choice(["bf16", "fp16"])
    while True:
        if op == "checkpoint":
            case = {"op": op, "tokens": _spread(rng, 1, 32768), "inner": _spread(rng, 16, 4096), "dtype": dtype}
        elif op in ("loss", "loss_step"):
            case = {"op": op, "tokens": _spread(rng, 1, 8192), "inner": _spread(rng, 16, 4096),
                    "vocab": _spread(rng, 3, 1000003), "ignored": rng.choice([0.0, 0.05, 0.33]), "dtype": dtype}
            if case["tokens"] * case["vocab"] > 1.2e9:  # the plain form keeps the logits
                continue
        else:
            case = {"op": op, "tokens": _spread(rng, 1, 16384), "inner": _spread(rng, 13, 4096),
                    "width": _spread(rng, 16, 12288), "act": rng.choice(["silu", "gelu", "relu", "identity"]),
                    "dtype": dtype}
        if work(case)["flops"] <= LARGEST:
            return case


def work(case):
    """Bytes: every input read once, every output written once (the 8-bit
    copy, which outlives the forward pass, written and read).  Flops: the
    matrix products.  The backward pass has X and the weights, so forming
    G = X Wg^T and U = X Wu^T belongs to it."""
    op, t, k = case["op"], case["tokens"], case["inner"]
    eight = t * (k + -(-k // GROUP))
    if op == "checkpoint":
        return {"bytes": 2 * t * k + 2 * eight + 2 * t * k, "flops": 3 * t * k}
    if op in ("loss", "loss_step"):
        v = case["vocab"]
        if op == "loss":
            return {"bytes": 2 * (t * k + v * k) + 12 * t, "flops": 2 * t * k * v}
        return {"bytes": 4 * (t * k + v * k) + 16 * t, "flops": 6 * t * k * v}
    f = case["width"]
    forward = {"bytes": 2 * (t * k + 2 * f * k + t * f), "flops": 4 * t * k * f}
    backward = {"bytes": 2 * (t * f + 2 * t * k + 4 * f * k), "flops": 12 * t * k * f}
    if op == "gated":
        return forward
    if op == "gated_backward":
        return backward
    return {"bytes": forward["bytes"] + backward["bytes"] - 2 * t * k + 2 * eight,
            "flops": forward["flops"] + backward["flops"]}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    t, k, op = case["tokens"], case["inner"], case["op"]

    def normal(*shape, std=1.0, dt=dtype):
        return (torch.randn(shape, generator=gen, device=dev, dtype=torch.float32) * std).to(dt)

    state = {"op": op, "x": normal(t, k)}
    if op == "checkpoint":
        # a few features a hundred times as large, as activations have them
        wide = torch.rand(k, generator=gen, device=dev) < 0.01
        state["x"] = torch.where(wide, state["x"] * 100, state["x"])
    elif op in ("loss", "loss_step"):
        v = case["vocab"]
        state["w"] = normal(v, k, std=2.0 / math.sqrt(k))
        # targets by popularity: the lower the index the more often
        u = torch.rand(t, generator=gen, device=dev, dtype=torch.float64)
        target = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        left_out = torch.rand(t, generator=gen, device=dev) < case["ignored"]
        state["target"] = torch.where(left_out, torch.full_like(target, IGNORE), target)
        if op == "loss_step":
            # the gradient of a weighted mean, times the loss scale that 16-bit floats of a short range need
            scale = 4096.0 if case["dtype"] == "fp16" else 1.0
            state["dloss"] = (0.5 + torch.rand(t, generator=gen, device=dev)) * (scale / t)
    else:
        f = case["width"]
        state["act"] = case["act"]
        state["w_gate"] = normal(f, k, std=1.0 / math.sqrt(k))
        state["w_up"] = normal(f, k, std=1.0 / math.sqrt(k))
        if op != "gated":
            state["dh"] = normal(t, f)
    return state


# ------------------------------------------------------------------ the operators
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from helrm_b200 import training

    op, x = state["op"], state["x"]
    if op == "gated":
        return training.gated_forward(x, state["w_gate"], state["w_up"], state["act"])
    if op == "gated_backward":
        dx, dwg, dwu = training.gated_backward(state["dh"], x, state["w_gate"], state["w_up"], state["act"])
        return {"dx": dx, "dw_gate": dwg, "dw_up": dwu}
    if op == "checkpoint":
        return training.unpack_checkpoint(training.pack_checkpoint(x))
    if op == "checkpointed":
        kept = training.pack_checkpoint(x)
        h = training.gated_forward(x, state["w_gate"], state["w_up"], state["act"])
        dx, dwg, dwu = training.gated_backward(state["dh"], kept, state["w_gate"], state["w_up"], state["act"])
        return {"h": h, "dx": dx, "dw_gate": dwg, "dw_up": dwu}
    loss, lse = training.vocabulary_loss_forward(x, state["w"], state["target"], ignore_index=IGNORE)
    if op == "loss":
        return loss
    dh, dw = training.vocabulary_loss_backward(state["dloss"], x, state["w"], state["target"], lse,
                                               ignore_index=IGNORE)
    return {"loss": loss, "dh": dh, "dw": dw}


def _plain(state):
    op, x = state["op"], state["x"]
    if op == "gated":
        return _plain_gated(x.float(), state).to(x.dtype)
    if op == "gated_backward":
        return _plain_gated_backward(x.float(), state)
    if op == "checkpoint":
        return _plain_checkpoint(x).to(x.dtype)
    if op == "checkpointed":
        h = _plain_gated(x.float(), state).to(x.dtype)
        return {"h": h, **_plain_gated_backward(_plain_checkpoint(x), state)}
    return _plain_loss(state, op == "loss_step")


def _act(g, act):
    """act(g) and its derivative."""
    if act == "identity":
        return g, torch.ones_like(g)
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    s = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * s, s + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_gated(x, state):
    g = x @ state["w_gate"].float().T
    u = x @ state["w_up"].float().T
    return _act(g, state["act"])[0] * u


def _plain_gated_backward(x, state):
    dtype = state["w_gate"].dtype
    wg, wu, dh = state["w_gate"].float(), state["w_up"].float(), state["dh"].float()
    a, d = _act(x @ wg.T, state["act"])
    du = dh * a
    dg = dh * (x @ wu.T) * d
    return {"dx": (dg @ wg + du @ wu).to(dtype), "dw_gate": (dg.T @ x).to(dtype), "dw_up": (du.T @ x).to(dtype)}


def _plain_checkpoint(x):
    """The 32-bit values that the 8-bit copy of x stands for: the least
    power of two s with max |x| <= 127 s in the group (from 2^-126 on, or
    2^-24 for fp16) and whole numbers of s, halves to even."""
    t, k = x.shape
    pad = -k % GROUP
    v = x.float()
    if pad:
        v = torch.cat([v, v.new_zeros(t, pad)], dim=1)
    v = v.view(t, -1, GROUP)
    m, e = torch.frexp(v.abs().amax(dim=2, keepdim=True))
    e = torch.where(m * 128 > 127, e - 6, e - 7)
    least, most, top = (-24, 10, 63.0) if x.dtype == torch.float16 else (-126, 122, 63.0)
    e = torch.where(m > 0, e, torch.full_like(e, least)).clamp(min=least)
    s = ((e + 127).to(torch.int32) << 23).view(torch.float32)
    q = torch.round(v / s)
    q = torch.where(e == most, q.clamp(-top, top), q)
    return (q * s).reshape(t, -1)[:, :k]


def _plain_loss(state, step):
    x, w, target = state["x"].float(), state["w"].float(), state["target"]
    valid = target != IGNORE
    t = torch.where(valid, target, torch.zeros_like(target))[:, None]
    z = x @ w.T
    top = z.amax(dim=1, keepdim=True)
    at = z.gather(1, t)
    z = torch.exp(z - top)
    s = z.sum(dim=1, keepdim=True)
    loss = torch.where(valid, (top + torch.log(s) - at)[:, 0], torch.zeros_like(s[:, 0]))
    if not step:
        return loss
    coef = torch.where(valid, state["dloss"], torch.zeros_like(state["dloss"]))[:, None]
    z = z * (coef / s)
    z.scatter_add_(1, t, -coef)
    return {"loss": loss, "dh": (z @ w).to(state["x"].dtype), "dw": (z.T @ x).to(state["w"].dtype)}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """run()'s outputs in 64 bits, the gradients by automatic differentiation."""
    state = prepare(case, seed)
    op, x = state["op"], state["x"].double()
    if op == "checkpoint":
        return _exact_checkpoint(state["x"])
    if op in ("loss", "loss_step"):
        return _exact_loss(state, op == "loss_step")
    act = {"identity": lambda v: v, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu}[state["act"]]
    wg, wu = (state[n].double().requires_grad_(op != "gated") for n in ("w_gate", "w_up"))
    block = torch.nn.functional.linear

    def forward(v):
        return act(block(v, wg)) * block(v, wu)

    if op == "gated":
        return forward(x)
    kept = (_exact_checkpoint(state["x"]) if op == "checkpointed" else x).detach().requires_grad_(True)
    dx, dwg, dwu = torch.autograd.grad(forward(kept), (kept, wg, wu), state["dh"].double())
    out = {"dx": dx, "dw_gate": dwg, "dw_up": dwu}
    if op == "checkpointed":
        with torch.no_grad():
            out["h"] = forward(x)
    return out


def _two_to(e):
    return (e + 1023 << 52).view(torch.float64)


def _exact_checkpoint(x):
    half = x.dtype == torch.float16
    largest = torch.finfo(x.dtype).max
    parts = []
    for part in x.double().split(GROUP, dim=1):
        top = part.abs().amax(dim=1, keepdim=True)
        e = torch.ceil(torch.log2(top)).clamp(-1000, 1000).long() - 7
        e = torch.where(127 * _two_to(e) < top, e + 1, e)
        s = _two_to(e.clamp(min=-24 if half else -126))
        q = torch.round(part / s)
        fits = torch.floor(largest / s)  # the last whole number whose product the type holds
        parts.append(torch.minimum(torch.maximum(q, -fits), fits) * s)
    return torch.cat(parts, dim=1)


def _exact_loss(state, step):
    w = state["w"].double().requires_grad_(step)
    rows = max(1, int(1.5e8 // w.shape[0]))
    losses, dhs, dw = [], [], None
    for i in range(0, state["x"].shape[0], rows):
        h = state["x"][i:i + rows].double().requires_grad_(step)
        loss = torch.nn.functional.cross_entropy(torch.nn.functional.linear(h, w), state["target"][i:i + rows],
                                                 ignore_index=IGNORE, reduction="none")
        losses.append(loss.detach())
        if step:
            dh, part = torch.autograd.grad(loss, (h, w), state["dloss"][i:i + rows].double())
            dhs.append(dh)
            dw = part if dw is None else dw.add_(part)
        del loss
    loss = torch.cat(losses)
    return {"loss": loss, "dh": torch.cat(dhs), "dw": dw} if step else loss
