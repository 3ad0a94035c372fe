"""Operators that train, in the clear, the weights the encrypted forward evaluates.

The backend evaluates a recommendation model's weights on ciphertexts; these
are the operators that find them, on torch tensors of a B200:

* :func:`gated_feed_forward`, ``act(x Wg^T) * (x Wu^T)``, with its gradients.
  With ``activation="identity"`` the block is two linear transforms and one
  ciphertext product, so what was trained runs encrypted as it is;
* 8-bit checkpoints of activations (:func:`pack_checkpoint`), from which the
  block's backward pass can start (``checkpoint=True``);
* :func:`vocabulary_cross_entropy`, the softmax cross entropy of ``h W^T``
  over the rows of ``W``, with its gradients, without the logits in memory.

Each is differentiable, once and in reverse; the ``*_forward`` /
``*_backward`` functions under them are the single passes, which record no
gradient: their results require none, whatever their inputs do.

Tensors are 16-bit floats (``torch.float16`` or ``torch.bfloat16``, one type
per call) of one CUDA device, any leading dimensions; work goes to the
device's current torch stream, workspaces come from torch's allocator, and
nothing but :func:`synchronize` waits.  Losses and sums are in 32 bits; the
gradients by the block's projections and by the logits are rounded to the
16-bit type once, as operands of the products that follow, which makes a
result's error 1.3 to 1.4 times that of its own rounding.  Failures raise like
the backend's: ``ValueError`` for arguments, ``RuntimeError`` for CUDA.
"""
from __future__ import annotations

import ctypes
import operator
from typing import NamedTuple

import torch

from . import _capi

GROUP = 32  # features that share a scale in a checkpoint
ACTIVATIONS = {"identity": 0, "relu": 1, "silu": 2, "gelu": 3}
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


class Checkpoint(NamedTuple):
    """An activation in 8 bits: ``q * 2^(e - 127)`` by groups of 32 features
    (``q`` [rows, 32 groups], ``e`` [rows, groups]); read it back with
    :func:`unpack_checkpoint`."""
    q: torch.Tensor
    e: torch.Tensor
    shape: tuple
    dtype: torch.dtype


# ------------------------------------------------------------------ arguments
def _matrix(t, name: str, cols: int | None = None):
    """t as rows of one pitch (a view where the strides allow it)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} is not a tensor")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} is {t.dtype}: the training operators take torch.float16 or torch.bfloat16")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: the training operators run on a CUDA device only")
    shape = t.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"{name} has no features (shape {tuple(shape)})")
    if cols is not None and shape[-1] != cols:
        raise ValueError(f"{name} has {shape[-1]} features where {cols} are expected")
    m = t if len(shape) == 2 else t.reshape(-1, shape[-1])
    if m.is_contiguous():
        return m
    rows, cols = m.shape
    if m.stride(1) != 1 and cols > 1 or rows > 1 and m.stride(0) < cols:
        m = m.contiguous()
    return m


def _weight(t, name: str, cols: int):
    if isinstance(t, torch.Tensor) and t.dim() != 2:
        raise ValueError(f"{name} is not a matrix (shape {tuple(t.shape)})")
    return _matrix(t, name, cols)


def _pitch(m) -> int:
    return m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _same(first, **others):
    for name, t in others.items():
        if t.dtype != first.dtype:
            raise ValueError(f"{name} is {t.dtype}, not {first.dtype}")
        if t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, not {first.device}")


def _activation(name: str) -> int:
    if not isinstance(name, str) or name not in ACTIVATIONS:
        raise ValueError(f"activation {name!r} is none of {sorted(ACTIVATIONS)}")
    return ACTIVATIONS[name]


_entries: dict = {}
_plans: dict = {}  # what a call with these types, shapes and strides comes to
_NOTHING = ctypes.byref(ctypes.c_size_t(0))


def _entry(name: str):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_capi.load(), name)
    return fn


_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # absent where torch has no CUDA


class _Plan:
    """The checked form of a call: the entry's leading arguments, the row
    pitches of its matrices, what it returns, and the workspace it needs by
    which addresses are on 16-byte boundaries."""
    __slots__ = ("head", "pitches", "out", "needs")

    def __init__(self, head, pitches, out):
        self.head, self.pitches, self.out, self.needs = head, pitches, out, {}


class _Out:
    """A dense result (with its strides at hand torch allocates it fastest)."""
    __slots__ = ("shape", "strides", "dtype", "device")

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.device = tuple(shape), dtype, device
        n, strides = 1, []
        for d in reversed(self.shape):
            strides.insert(0, n)
            n *= max(1, d)
        self.strides = tuple(strides)

    def new(self):
        return torch.empty_strided(self.shape, self.strides, dtype=self.dtype, device=self.device)


def _remember(key, plan):
    if key is None:  # of something that cannot be a key, a shape in a list
        return
    if len(_plans) > 4096:
        _plans.clear()
    _plans[key] = plan


def _run(fn, like, needs, odd, *args):
    """One entry point that takes a workspace, on the current stream of
    like's device.  needs: the bytes it takes, by odd."""
    need = needs.get(odd)
    if need is None:
        n = ctypes.c_size_t(0)
        _capi.check(fn(*args, None, ctypes.byref(n), 0))
        need = needs[odd] = n.value
    if need:
        ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=like.device)
        rc = fn(*args, ws.data_ptr(), ctypes.byref(ctypes.c_size_t(need)), _stream(args[0]))
    else:  # any aligned address will do
        rc = fn(*args, 256, _NOTHING, _stream(args[0]))
    if rc:
        _capi.check(rc)


def synchronize(device=None):
    """Waits for the current stream of the device (the current one).  Raises
    RuntimeError if a kernel of a call since the last report gave up waiting (a
    hardware failure), as the next call on that device would; a program's last
    call has no next one."""
    with torch.cuda.device(device):
        index = torch.cuda.current_device()
    _capi.check(_entry("helrm_TrainingSynchronize")(index, _stream(index)))


# ------------------------------------------------------------------ the gated block
def gated_forward(x, w_gate, w_up, activation: str = "silu"):
    """act(x w_gate^T) * (x w_up^T), in one kernel; x [..., inner], weights
    [width, inner], the result [..., width]."""
    try:
        key = (activation, x.dtype, x.device, x.shape, x.stride(), w_gate.dtype, w_gate.device, w_gate.shape,
               w_gate.stride(), w_up.dtype, w_up.device, w_up.shape, w_up.stride())
        plan = _plans.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        act = _activation(activation)
        xm = _matrix(x, "x")
        inner = xm.shape[1]
        wg, wu = _weight(w_gate, "w_gate", inner), _weight(w_up, "w_up", inner)
        _same(xm, w_gate=wg, w_up=wu)
        if wg.shape != wu.shape:
            raise ValueError(f"w_gate {tuple(wg.shape)} and w_up {tuple(wu.shape)} differ in shape")
        width = wg.shape[0]
        if width < 1:
            raise ValueError("the weights have no rows")
        plan = _Plan((x.device.index, _DTYPES[x.dtype], act, xm.shape[0], inner, width),
                     (_pitch(xm), _pitch(wg), _pitch(wu)), _Out(x.shape[:-1] + (width,), x.dtype, x.device))
        if xm.data_ptr() == x.data_ptr() and wg is w_gate and wu is w_up:
            _remember(key, plan)
        x, w_gate, w_up = xm, wg, wu  # the copies, where the strides asked for some
    o = plan.out
    h = torch.empty_strided(o.shape, o.strides, dtype=o.dtype, device=o.device)
    px, pg, pu = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr()
    lx, lg, lu = plan.pitches
    _run(_entry("helrm_GatedForward"), x, plan.needs, (px & 15, pg & 15, pu & 15), *plan.head, px, lx, pg, lg, pu, lu,
         h.data_ptr())
    return h


def gated_backward(dh, x, w_gate, w_up, activation: str = "silu", needs=(True, True, True)):
    """(dx, dw_gate, dw_up) from dh, the gradient by gated_forward's result.
    x is the block's input or its Checkpoint; the projections are formed
    again.  needs: which of the three are wanted (None in their place)."""
    kept = isinstance(x, Checkpoint)
    try:
        xk = (x.q.dtype, x.q.device, x.q.shape, x.q.stride(), x.e.dtype, x.e.device, x.e.shape, x.e.stride(), x.shape,
              x.dtype, x.q.data_ptr() & 15) if kept else (x.dtype, x.device, x.shape, x.stride())
        key = (activation, tuple(needs), xk, dh.dtype, dh.device, dh.shape, dh.stride(), w_gate.dtype, w_gate.device,
               w_gate.shape, w_gate.stride(), w_up.dtype, w_up.device, w_up.shape, w_up.stride())
        plan = _plans.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        act = _activation(activation)
        dhm = _matrix(dh, "dh")
        if kept:
            _check_checkpoint(x)
            xm, shape, inner, pitch = x, tuple(x.shape), x.shape[-1], x.shape[-1]
            if x.dtype != dhm.dtype or x.q.device != dhm.device:
                raise ValueError(f"the checkpoint is {x.dtype} on {x.q.device}, dh {dhm.dtype} on {dhm.device}")
        else:
            xm = _matrix(x, "x")
            shape, inner, pitch = tuple(x.shape), xm.shape[1], _pitch(xm)
            _same(dhm, x=xm)
        wg, wu = _weight(w_gate, "w_gate", inner), _weight(w_up, "w_up", inner)
        _same(dhm, w_gate=wg, w_up=wu)
        if wg.shape != wu.shape:
            raise ValueError(f"w_gate {tuple(wg.shape)} and w_up {tuple(wu.shape)} differ in shape")
        tokens, width = dhm.shape
        if tuple(dh.shape) != shape[:-1] + (wg.shape[0],):
            raise ValueError(f"dh has shape {tuple(dh.shape)}, the block's result {shape[:-1] + (wg.shape[0],)}")
        plan = _Plan((dh.device.index, _DTYPES[dh.dtype], act, tokens, inner, width),
                     (_pitch(dhm), pitch, _pitch(wg), _pitch(wu)),
                     (_Out(shape, dh.dtype, dh.device), _Out((width, inner), dh.dtype, dh.device)))
        if (dhm.data_ptr() == dh.data_ptr() and (kept or xm.data_ptr() == x.data_ptr()) and wg is w_gate
                and wu is w_up):
            _remember(key, plan)
        dh, x, w_gate, w_up = dhm, xm, wg, wu  # the copies, where the strides asked for some
    out_x, out_w = plan.out
    dx = out_x.new() if needs[0] else None
    dwg = out_w.new() if needs[1] else None
    dwu = out_w.new() if needs[2] else None
    if any(needs):
        ld, lx, lg, lu = plan.pitches
        pd, pg, pu = dh.data_ptr(), w_gate.data_ptr(), w_up.data_ptr()
        px, pq, pe = (None, x.q.data_ptr(), x.e.data_ptr()) if kept else (x.data_ptr(), None, None)
        _run(_entry("helrm_GatedBackward"), dh, plan.needs, ((px or 0) & 15, pg & 15, pu & 15), *plan.head, pd, ld, px, lx, pq,
             pe, pg, lg, pu, lu, None if dx is None else dx.data_ptr(), None if dwg is None else dwg.data_ptr(),
             None if dwu is None else dwu.data_ptr())
    return dx, dwg, dwu


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation, checkpoint):
        ctx.activation, ctx.kept = activation, None
        if checkpoint:
            c = pack_checkpoint(x)
            ctx.kept = (c.shape, c.dtype)
            ctx.save_for_backward(c.q, c.e, w_gate, w_up)
        else:
            ctx.save_for_backward(x, w_gate, w_up)
        return gated_forward(x, w_gate, w_up, activation)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        *x, w_gate, w_up = ctx.saved_tensors
        x = Checkpoint(*x, *ctx.kept) if ctx.kept else x[0]
        return (*gated_backward(dh, x, w_gate, w_up, ctx.activation, ctx.needs_input_grad[:3]), None, None)


def gated_feed_forward(x, w_gate, w_up, activation: str = "silu", checkpoint: bool = False):
    """act(x w_gate^T) * (x w_up^T), differentiable.  The backward pass needs
    x alone; with checkpoint it keeps x in 8 bits (33 bytes for 32 features of a
    row, or a part of 32: half the memory of long rows, more than all of it for
    16 features or fewer) and its gradients are those at the values the 8 bits
    stand for.  Where no gradient is recorded nothing is kept."""
    if checkpoint:
        checkpoint = torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in (x, w_gate, w_up))
    return _GatedFeedForward.apply(x, w_gate, w_up, activation, checkpoint)


# ------------------------------------------------------------------ 8-bit checkpoints
def _check_checkpoint(c):
    if (not isinstance(c.q, torch.Tensor) or not isinstance(c.e, torch.Tensor) or not isinstance(c.dtype, torch.dtype)
            or not isinstance(c.shape, (tuple, list)) or not c.shape or not all(isinstance(n, int) for n in c.shape)):
        raise ValueError("not a checkpoint that pack_checkpoint returned")
    rows = 1
    for n in c.shape[:-1]:
        rows *= n
    groups = -(-c.shape[-1] // GROUP)
    if (c.dtype not in _DTYPES or c.q.dtype != torch.int8 or c.e.dtype != torch.uint8
            or tuple(c.q.shape) != (rows, GROUP * groups) or tuple(c.e.shape) != (rows, groups)
            or not c.q.is_contiguous() or not c.e.is_contiguous() or not c.q.is_cuda or c.e.device != c.q.device
            or c.q.data_ptr() % 16):
        raise ValueError("not a checkpoint that pack_checkpoint returned")
    return rows


def pack_checkpoint(x) -> Checkpoint:
    """x [..., features] in 8 bits: groups of 32 features share the least
    power of two s with max |x| <= 127 s, the values are whole numbers of s
    (rounded, halves to even).  A group that holds an infinity or a NaN reads
    back as NaN."""
    try:
        key = ("pack", x.dtype, x.device, x.shape, x.stride())
        plan = _plans.get(key)
    except AttributeError:
        key = plan = None
    if plan is None:
        m = _matrix(x, "x")
        rows, cols = m.shape
        groups = -(-cols // GROUP)
        plan = _Plan((x.device.index, _DTYPES[x.dtype], rows, cols), _pitch(m),
                     (_Out((rows, GROUP * groups), torch.int8, x.device), _Out((rows, groups), torch.uint8, x.device),
                      tuple(x.shape), x.dtype))
        if m.data_ptr() == x.data_ptr():
            _remember(key, plan)
        x = m
    out_q, out_e, shape, dtype = plan.out
    q, e = out_q.new(), out_e.new()
    rc = _entry("helrm_PackCheckpoint")(*plan.head, x.data_ptr(), plan.pitches, q.data_ptr(), e.data_ptr(),
                                        _stream(plan.head[0]))
    if rc:
        _capi.check(rc)
    return Checkpoint(q, e, shape, dtype)


def unpack_checkpoint(c: Checkpoint):
    """The tensor a checkpoint stands for, exact in its 16-bit type."""
    if not isinstance(c, Checkpoint):
        raise ValueError("not a checkpoint that pack_checkpoint returned")
    q, e, shape, dtype = c
    try:
        key = ("unpack", q.dtype, q.device, q.shape, q.stride(), e.dtype, e.device, e.shape, e.stride(), shape, dtype,
               q.data_ptr() & 15)
        plan = _plans.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        rows = _check_checkpoint(c)
        plan = _Plan((q.device.index, _DTYPES[dtype], rows, shape[-1]), None, _Out(shape, dtype, q.device))
        _remember(key, plan)
    x = plan.out.new()
    rc = _entry("helrm_UnpackCheckpoint")(*plan.head, q.data_ptr(), e.data_ptr(), x.data_ptr(),
                                          _stream(plan.head[0]))
    if rc:
        _capi.check(rc)
    return x


# ------------------------------------------------------------------ the loss
def _targets(targets, lead, dev):
    if not isinstance(targets, torch.Tensor) or targets.dtype not in (torch.int64, torch.int32):
        raise ValueError("targets is not an int64 or int32 tensor")
    if targets.device != dev:
        raise ValueError(f"targets is on {targets.device}, not {dev}")
    if tuple(targets.shape) != tuple(lead):
        raise ValueError(f"targets has shape {tuple(targets.shape)}, the rows of h {tuple(lead)}")
    return targets.to(torch.int64).contiguous()


def _ignored(index) -> int:
    try:
        index = operator.index(index)
    except TypeError:
        raise ValueError(f"ignore_index {index!r} is no whole number") from None
    if not -2 ** 63 <= index < 2 ** 63:
        raise ValueError(f"ignore_index {index} does not fit 64 bits")
    return index


def _floats(t, name: str, like: _Out):
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != like.device
            or t.shape != like.shape):
        raise ValueError(f"{name} is not a float32 tensor of shape {like.shape} on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _loss_call(h, w, targets):
    """(h, w, targets as the entries take them, the plan)"""
    try:
        key = ("loss", h.dtype, h.device, h.shape, h.stride(), w.dtype, w.device, w.shape, w.stride(), targets.dtype,
               targets.device, targets.shape)
        plan = _plans.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        hm = _matrix(h, "h")
        wm = _weight(w, "w", hm.shape[1])
        _same(hm, w=wm)
        if wm.shape[0] < 1:
            raise ValueError("w has no rows")
        lead = h.shape[:-1]
        t = _targets(targets, lead, h.device)
        plan = _Plan((h.device.index, _DTYPES[h.dtype], hm.shape[0], hm.shape[1], wm.shape[0]),
                     (_pitch(hm), _pitch(wm)),
                     (_Out(lead, torch.float32, h.device), _Out(lead + (2,), torch.float32, h.device),
                      _Out(h.shape, h.dtype, h.device), _Out(wm.shape, h.dtype, h.device)))
        if hm.data_ptr() == h.data_ptr() and wm is w:
            _remember(key, plan)
        return hm, wm, t, plan
    if targets.dtype != torch.int64 or not targets.is_contiguous():
        targets = targets.to(torch.int64).contiguous()
    return h, w, targets, plan


def vocabulary_loss_forward(h, w, targets, ignore_index: int = -100):
    """(loss, lse), float32: for each row loss = lse - h . w[target] with
    lse = log sum_j exp(h . w[j]), kept as the sum of two numbers, lse [..., 2]:
    the largest logit and the log of the sum relative to it.  h [..., inner],
    w [vocab, inner], targets [...].  Rows whose target is ignore_index have
    loss 0, other targets outside the vocabulary NaN."""
    ignore_index = _ignored(ignore_index)
    h, w, t, plan = _loss_call(h, w, targets)
    loss, lse = plan.out[0].new(), plan.out[1].new()
    ph, pw = h.data_ptr(), w.data_ptr()
    _run(_entry("helrm_VocabularyLossForward"), h, plan.needs, (ph & 15, pw & 15), *plan.head, ph, plan.pitches[0], pw,
         plan.pitches[1], t.data_ptr(), ignore_index, loss.data_ptr(), lse.data_ptr())
    return loss, lse


def vocabulary_loss_backward(dloss, h, w, targets, lse, ignore_index: int = -100, needs=(True, True)):
    """(dh, dw) from dloss [...] (float32) and vocabulary_loss_forward's lse.
    needs: which of the two are wanted (None in their place)."""
    ignore_index = _ignored(ignore_index)
    h, w, t, plan = _loss_call(h, w, targets)
    out_loss, out_lse, out_h, out_w = plan.out
    g, l = _floats(dloss, "dloss", out_loss), _floats(lse, "lse", out_lse)
    if l.data_ptr() & 7:  # read in pairs
        l = l.clone()
    dh = out_h.new() if needs[0] else None
    dw = out_w.new() if needs[1] else None
    if any(needs):
        ph, pw = h.data_ptr(), w.data_ptr()
        _run(_entry("helrm_VocabularyLossBackward"), h, plan.needs, (ph & 15, pw & 15, bool(needs[0]), bool(needs[1])),
             *plan.head, g.data_ptr(), ph, plan.pitches[0], pw, plan.pitches[1], t.data_ptr(), l.data_ptr(),
             ignore_index, None if dh is None else dh.data_ptr(), None if dw is None else dw.data_ptr())
    return dh, dw


class _VocabularyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, targets, ignore_index):
        loss, lse = vocabulary_loss_forward(h, w, targets, ignore_index)
        ctx.ignore_index = ignore_index
        ctx.save_for_backward(h, w, targets, lse)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        h, w, targets, lse = ctx.saved_tensors
        return (*vocabulary_loss_backward(dloss, h, w, targets, lse, ctx.ignore_index, ctx.needs_input_grad[:2]), None,
                None)


def vocabulary_cross_entropy(h, w, targets, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of h w^T against targets, differentiable in h and
    w, without the logits in memory.  reduction: "mean" over the rows that
    are not ignored, "sum", or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction {reduction!r} is none of 'mean', 'sum', 'none'")
    ignore_index = _ignored(ignore_index)
    loss = _VocabularyLoss.apply(h, w, targets, ignore_index)
    if reduction == "none":
        return loss
    total = loss.sum()
    return total if reduction == "sum" else total / (targets != ignore_index).sum()
