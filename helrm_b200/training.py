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

Each is differentiable; the ``*_forward`` / ``*_backward`` functions under
them are the single passes.  Tensors are 16-bit floats (``torch.float16`` or
``torch.bfloat16``, one type per call) of one CUDA device, any leading
dimensions; work goes to the device's current torch stream, workspaces come
from torch's allocator, and nothing synchronises.  Losses and sums are in 32
bits.  Failures raise like the backend's: ``ValueError`` for arguments,
``RuntimeError`` for CUDA.
"""
from __future__ import annotations

import ctypes
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


def _place(m):
    """(address, row pitch)"""
    return m.data_ptr(), m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _same(first, **others):
    for name, t in others.items():
        if t.dtype != first.dtype:
            raise ValueError(f"{name} is {t.dtype}, not {first.dtype}")
        if t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, not {first.device}")


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation {name!r} is none of {sorted(ACTIVATIONS)}")
    return ACTIVATIONS[name]


_entries: dict = {}
_workspaces: dict = {}  # bytes an entry needs, by its sizes, pitches and alignments


def _entry(name: str):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_capi.load(), name)
    return fn


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _run(name: str, dev, sizes, *args):
    """One entry point that takes a workspace, on dev's current stream.
    sizes: what the workspace depends on."""
    fn = _entry(name)
    need = _workspaces.get(key := (name, sizes))
    if need is None:
        if len(_workspaces) > 4096:
            _workspaces.clear()
        n = ctypes.c_size_t(0)
        _capi.check(fn(*args, None, ctypes.byref(n), 0))
        need = _workspaces[key] = n.value
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        rc = fn(*args, ws.data_ptr(), ctypes.byref(ctypes.c_size_t(need)), _stream(dev.index))
    else:  # any aligned address will do
        rc = fn(*args, 256, ctypes.byref(ctypes.c_size_t(0)), _stream(dev.index))
    if rc:
        _capi.check(rc)


# ------------------------------------------------------------------ the gated block
def gated_forward(x, w_gate, w_up, activation: str = "silu"):
    """act(x w_gate^T) * (x w_up^T), in one kernel; x [..., inner], weights
    [width, inner], the result [..., width]."""
    act = _activation(activation)
    xm = _matrix(x, "x")
    inner = xm.shape[1]
    wg, wu = _weight(w_gate, "w_gate", inner), _weight(w_up, "w_up", inner)
    _same(xm, w_gate=wg, w_up=wu)
    if wg.shape != wu.shape:
        raise ValueError(f"w_gate {tuple(wg.shape)} and w_up {tuple(wu.shape)} differ in shape")
    tokens, width = xm.shape[0], wg.shape[0]
    if width < 1:
        raise ValueError("the weights have no rows")
    h = torch.empty(x.shape[:-1] + (width,), dtype=x.dtype, device=x.device)
    dev = x.device
    px, lx, pg, lg, pu, lu = *_place(xm), *_place(wg), *_place(wu)
    _run("helrm_GatedForward", dev, (tokens, inner, width, px % 16, lx, pg % 16, lg, pu % 16, lu), dev.index,
         _DTYPES[x.dtype], act, tokens, inner, width, px, lx, pg, lg, pu, lu, h.data_ptr())
    return h


def gated_backward(dh, x, w_gate, w_up, activation: str = "silu", needs=(True, True, True)):
    """(dx, dw_gate, dw_up) from dh, the gradient by gated_forward's result.
    x is the block's input or its Checkpoint; the projections are formed
    again.  needs: which of the three are wanted (None in their place)."""
    act = _activation(activation)
    dhm = _matrix(dh, "dh")
    kept = isinstance(x, Checkpoint)
    if kept:
        shape, inner = tuple(x.shape), x.shape[-1]
        _check_checkpoint(x)
        if x.dtype != dhm.dtype or x.q.device != dhm.device:
            raise ValueError(f"the checkpoint is {x.dtype} on {x.q.device}, dh {dhm.dtype} on {dhm.device}")
        xm = None
    else:
        xm = _matrix(x, "x")
        shape, inner = tuple(x.shape), xm.shape[1]
        _same(dhm, x=xm)
    wg, wu = _weight(w_gate, "w_gate", inner), _weight(w_up, "w_up", inner)
    _same(dhm, w_gate=wg, w_up=wu)
    if wg.shape != wu.shape:
        raise ValueError(f"w_gate {tuple(wg.shape)} and w_up {tuple(wu.shape)} differ in shape")
    tokens, width = dhm.shape
    if tuple(dh.shape) != shape[:-1] + (wg.shape[0],):
        raise ValueError(f"dh has shape {tuple(dh.shape)}, the block's result {shape[:-1] + (wg.shape[0],)}")
    like = dict(dtype=dh.dtype, device=dh.device)
    dx = torch.empty(shape, **like) if needs[0] else None
    dwg = torch.empty((width, inner), **like) if needs[1] else None
    dwu = torch.empty((width, inner), **like) if needs[2] else None
    if any(needs):
        dev = dh.device
        px, lx = (0, inner) if kept else _place(xm)
        pd, ld, pg, lg, pu, lu = *_place(dhm), *_place(wg), *_place(wu)
        _run("helrm_GatedBackward", dev,
             (tokens, inner, width, kept, px % 16, lx, pg % 16, lg, pu % 16, lu, *(bool(n) for n in needs)),
             dev.index, _DTYPES[dh.dtype], act, tokens, inner, width, pd, ld, px or None, lx,
             x.q.data_ptr() if kept else None, x.e.data_ptr() if kept else None, pg, lg, pu, lu,
             *(None if t is None else t.data_ptr() for t in (dx, dwg, dwu)))
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
    x alone; with checkpoint it keeps x in 8 bits (half the memory) and its
    gradients are those at the values the 8 bits stand for."""
    return _GatedFeedForward.apply(x, w_gate, w_up, activation, checkpoint)


# ------------------------------------------------------------------ 8-bit checkpoints
def _check_checkpoint(c):
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
    m = _matrix(x, "x")
    rows, cols = m.shape
    groups = -(-cols // GROUP)
    q = torch.empty((rows, GROUP * groups), dtype=torch.int8, device=x.device)
    e = torch.empty((rows, groups), dtype=torch.uint8, device=x.device)
    dev = x.device.index
    rc = _entry("helrm_PackCheckpoint")(dev, _DTYPES[x.dtype], rows, cols, *_place(m), q.data_ptr(), e.data_ptr(),
                                        _stream(dev))
    if rc:
        _capi.check(rc)
    return Checkpoint(q, e, tuple(x.shape), x.dtype)


def unpack_checkpoint(c: Checkpoint):
    """The tensor a checkpoint stands for, exact in its 16-bit type."""
    if not isinstance(c, Checkpoint):
        raise ValueError("not a checkpoint that pack_checkpoint returned")
    rows = _check_checkpoint(c)
    x = torch.empty(c.shape, dtype=c.dtype, device=c.q.device)
    dev = x.device.index
    rc = _entry("helrm_UnpackCheckpoint")(dev, _DTYPES[c.dtype], rows, c.shape[-1], c.q.data_ptr(), c.e.data_ptr(),
                                          x.data_ptr(), _stream(dev))
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


def _floats(t, name: str, lead, dev):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != dev or tuple(t.shape) != tuple(lead):
        raise ValueError(f"{name} is not a float32 tensor of shape {tuple(lead)} on {dev}")
    return t.contiguous()


def vocabulary_loss_forward(h, w, targets, ignore_index: int = -100):
    """(loss, lse), float32: for each row loss = lse - h . w[target] with
    lse = log sum_j exp(h . w[j]), kept as the sum of two numbers, lse [..., 2]:
    the largest logit and the log of the sum relative to it.  h [..., inner],
    w [vocab, inner], targets [...].  Rows whose target is ignore_index have
    loss 0, other targets outside the vocabulary NaN."""
    hm = _matrix(h, "h")
    wm = _weight(w, "w", hm.shape[1])
    _same(hm, w=wm)
    if wm.shape[0] < 1:
        raise ValueError("w has no rows")
    t = _targets(targets, h.shape[:-1], h.device)
    loss = torch.empty(h.shape[:-1], dtype=torch.float32, device=h.device)
    lse = torch.empty(h.shape[:-1] + (2,), dtype=torch.float32, device=h.device)
    dev, tokens, inner, vocab = h.device, hm.shape[0], hm.shape[1], wm.shape[0]
    ph, lh, pw, lw = *_place(hm), *_place(wm)
    _run("helrm_VocabularyLossForward", dev, (tokens, inner, vocab, ph % 16, lh, pw % 16, lw), dev.index,
         _DTYPES[h.dtype], tokens, inner, vocab, ph, lh, pw, lw, t.data_ptr(), int(ignore_index), loss.data_ptr(),
         lse.data_ptr())
    return loss, lse


def vocabulary_loss_backward(dloss, h, w, targets, lse, ignore_index: int = -100, needs=(True, True)):
    """(dh, dw) from dloss [...] (float32) and vocabulary_loss_forward's lse.
    needs: which of the two are wanted (None in their place)."""
    hm = _matrix(h, "h")
    wm = _weight(w, "w", hm.shape[1])
    _same(hm, w=wm)
    if wm.shape[0] < 1:
        raise ValueError("w has no rows")
    lead, dev = h.shape[:-1], h.device
    t = _targets(targets, lead, dev)
    g, l = _floats(dloss, "dloss", lead, dev), _floats(lse, "lse", lead + (2,), dev)
    dh = torch.empty(h.shape, dtype=h.dtype, device=dev) if needs[0] else None
    dw = torch.empty(wm.shape, dtype=h.dtype, device=dev) if needs[1] else None
    if any(needs):
        tokens, inner, vocab = hm.shape[0], hm.shape[1], wm.shape[0]
        ph, lh, pw, lw = *_place(hm), *_place(wm)
        _run("helrm_VocabularyLossBackward", dev,
             (h.dtype, tokens, inner, vocab, ph % 16, lh, pw % 16, lw, bool(needs[0]), bool(needs[1])), dev.index,
             _DTYPES[h.dtype], tokens, inner, vocab, g.data_ptr(), ph, lh, pw, lw, t.data_ptr(), l.data_ptr(),
             int(ignore_index), *(None if o is None else o.data_ptr() for o in (dh, dw)))
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
    loss = _VocabularyLoss.apply(h, w, targets, ignore_index)
    if reduction == "none":
        return loss
    total = loss.sum()
    return total if reduction == "sum" else total / (targets != ignore_index).sum()
