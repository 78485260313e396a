"""Products with packed weights on the device, without a decoded copy: one matrix times a few tokens (`matvec`), rows of a
table by their ids (`get_rows`), and a mixture-of-experts layer (`MoeLayer`).

A packed matrix is a uint8 CUDA tensor as it lies in a GGUF file: `rows` rows of `cols` elements, cols contiguous, of any
block type that `dequantize_slice` decodes (the reference decodes a tensor before it is used:
ggml-quants/src/lib.rs:135-147).  One of type F16 or BF16 may be a float16 or bfloat16 tensor instead.  As in `dequantize_slice` the destination comes first, the kernels run on torch's
current stream of the tensors' device (or on `stream`, a raw handle), and nothing is synchronized.  No gradients are
recorded: these are the products of serving.

    Q4K.matvec(y, w, x)           # y[t, r] = sum of W[r, c] x[t, c]
    Q4K.get_rows(y, w, ids)       # y[i] = row ids[i] of W
"""
import ctypes

import torch

from . import _lib
from ._lib import lib
from .quants import GGmlType, LengthMismatch, Indivisible, Unsupported, block_bytes, block_elems, check

_ELEM = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_IDS = {torch.int32: 26, torch.int64: 27}
_OWN = {1: torch.float16, 30: torch.bfloat16}      # element types that are block types too
_BLOCK = {}          # type id -> (elements, bytes of a block, the id as a plain number)
# A call takes about 5 us of the host's time, 3.9 of them for the launch; torch.cuda's own lookups would add 1.3.  Where this
# torch has the functions behind them, those are asked.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_matvec_device, _get_rows_device = lib.ggq_matvec_device, lib.ggq_get_rows_device


def _block(ty):
    b = _BLOCK.get(ty)
    if b is None:
        ty = int(ty)
        b = _BLOCK[ty] = (block_elems(ty), block_bytes(ty), ty)
    if b[0] == 0:
        raise Unsupported()
    return b


def _elem(t):
    k = _ELEM.get(t.dtype)
    if k is None:
        raise TypeError(f"unsupported element type {t.dtype}")
    return k


def _rows_of(t, what):
    """(tokens, width, stride between tokens) of a vector or of a matrix whose rows are contiguous."""
    shape = t.shape
    if len(shape) == 2:
        n, width = shape
        s0, s1 = t.stride()
    elif len(shape) == 1:
        n, (width,), (s1,) = 1, shape, t.stride()
        s0 = width
    else:
        raise ValueError(f"{what} must be a vector or a matrix")
    if s1 != 1 and width > 1:
        raise ValueError(f"the rows of {what} must be contiguous")
    return n, width, s0


def _device_of(first, *others):
    """The index of the one CUDA device that all tensors are on."""
    if not first.is_cuda:
        raise ValueError("tensors must be on the device")
    dev = first.get_device()
    for t in others:
        if not t.is_cuda or t.get_device() != dev:
            raise ValueError("tensors are on different devices")
    return dev


def _packed_bytes(ty, w):
    if w.dtype != torch.uint8 and w.dtype != _OWN.get(ty):
        raise TypeError(f"packed weights of type {ty} are uint8, not {w.dtype}")
    if not w.is_contiguous():
        raise ValueError("packed weights must be contiguous")
    return w.nbytes


def _call(dev, stream, fn, *args):
    """fn(*args, stream) with `dev` as the current device, on `stream` or on torch's current stream of that device."""
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return _call(dev, stream, fn, *args)
    if stream is None:
        stream = _current_stream(dev)
    status = fn(*args, stream)
    if status:
        check(status)


def matvec(ty, dst, w, x, stream=None):
    """dst[t, r] = sum over c of W[r, c] * x[t, c].

    `w`: packed rows of block type `ty`, dst.shape[-1] rows of x.shape[-1] elements.  `x` and `dst`: [tokens, ...] or one
    vector, float32, float16 or bfloat16 each, with contiguous rows and any stride between them.  Sums are held in 32 bits;
    see ggq_matvec_device in include/ggq.h for what is rounded before."""
    be, bb, ty = _block(ty)
    n, cols, xs = _rows_of(x, "x")
    m, rows, ys = _rows_of(dst, "dst")
    if n != m:
        raise LengthMismatch()
    if cols % be:
        raise Indivisible()
    if _packed_bytes(ty, w) != rows * (cols // be) * bb:
        raise LengthMismatch()
    _call(_device_of(dst, w, x), stream, _matvec_device, ty, rows, cols, w.data_ptr(), _elem(x), x.data_ptr(), xs, n,
          _elem(dst), dst.data_ptr(), ys)


def get_rows(ty, dst, w, ids, stream=None):
    """dst[i] = the decoded row ids[i] of the packed table `w` (dst.shape[-1] elements a row): token embeddings.

    `ids`: int32 or int64, contiguous; an id outside the table gives a row of zeros.  The values are those of
    `dequantize_slice`, bit for bit."""
    be, bb, ty = _block(ty)
    n, cols, ys = _rows_of(dst, "dst")
    kind = _IDS.get(ids.dtype)
    if kind is None:
        raise TypeError(f"unsupported id type {ids.dtype}")
    if not ids.is_contiguous():
        raise ValueError("ids must be contiguous")
    if ids.numel() != n:
        raise LengthMismatch()
    if cols % be:
        raise Indivisible()
    row = cols // be * bb
    size = _packed_bytes(ty, w)
    if row and size % row:
        raise LengthMismatch()
    _call(_device_of(dst, w, ids), stream, _get_rows_device, ty, size // row if row else 0, cols, w.data_ptr(), kind,
          ids.data_ptr(), n, _elem(dst), dst.data_ptr(), ys)


_GATING = {"softmax": 0, "sigmoid": 1}
_ACTIVATION = {"silu": 0, "gelu": 1}


class MoeLayer:
    """A mixture-of-experts layer with packed experts (ggq_moe_device): the feed-forward part of a model whose GGUF file
    holds ffn_gate_inp, ffn_gate_exps, ffn_up_exps and ffn_down_exps.

    `router`: [experts, hidden] float32, float16 or bfloat16 CUDA tensor.  `gate`, `up`, `down`: (block type, packed uint8
    tensor) of [experts][ff][hidden], the same and [experts][hidden][ff]; gate and up share one block type.  `gating`:
    "softmax" (over all experts) or "sigmoid"; `normalize`: the chosen experts' weights are divided by their sum; `scale`:
    a factor on the weights; `activation`: "silu" or "gelu" (tanh form).  The layer keeps its tensors alive."""

    def __init__(self, router, gate, up, down, *, hidden, ff, top_k, gating="softmax", normalize=True, scale=1.0, activation="silu"):
        (gt, gw), (ut, uw), (dt, dw) = gate, up, down
        if int(gt) != int(ut):
            raise Unsupported("gate and up must be of one block type")
        if gating not in _GATING or activation not in _ACTIVATION:
            raise ValueError("gating is softmax or sigmoid, activation is silu or gelu")
        if router.dim() != 2 or router.shape[1] != hidden or not router.is_contiguous():
            raise ValueError("router must be a contiguous [experts, hidden] matrix")
        experts = router.shape[0]
        (ue, ub, _), (de, db, _) = _block(ut), _block(dt)
        if hidden % ue or ff % de:
            raise Indivisible()
        for ty, w, size in ((gt, gw, experts * ff * (hidden // ue) * ub), (ut, uw, experts * ff * (hidden // ue) * ub), (dt, dw, experts * hidden * (ff // de) * db)):
            if _packed_bytes(int(ty), w) != size:
                raise LengthMismatch()
        self._dev = _device_of(router, gw, uw, dw)
        self._keep = (router, gw, uw, dw)
        self.hidden, self.ff, self.experts, self.top_k = hidden, ff, experts, top_k
        self._m = _lib.ggq_moe(_elem(router), int(ut), int(dt), 0, router.data_ptr(), gw.data_ptr(), uw.data_ptr(), dw.data_ptr(), hidden, ff,
                               experts, top_k, _GATING[gating], int(bool(normalize)), _ACTIVATION[activation], float(scale))
        self._ref = ctypes.byref(self._m)
        self._space = {}
        self.workspace_bytes(1)          # the description is checked here

    def workspace_bytes(self, tokens):
        n = self._space.get(tokens)
        if n is None:
            out = ctypes.c_size_t()
            check(lib.ggq_moe_workspace_bytes(self._ref, tokens, ctypes.byref(out)))
            n = self._space[tokens] = out.value
        return n

    def run(self, dst, x, ids=None, weights=None, stream=None):
        """dst[t] = the layer's output for x[t]; [tokens, hidden] or one vector each, float32, float16 or bfloat16, with
        contiguous rows.  `ids` (int32) and `weights` (float32), contiguous [tokens, top_k]: receive the experts chosen for
        each token, the largest logit first, and their weights.  At most 64 tokens a call.  The workspace comes from torch's
        allocator on the stream that the kernels run on, so calls on several streams do not share it."""
        n, cols, xs = _rows_of(x, "x")
        m, rows, ys = _rows_of(dst, "dst")
        if cols != self.hidden or rows != self.hidden or n != m:
            raise LengthMismatch()
        for t, dt in ((ids, torch.int32), (weights, torch.float32)):
            if t is not None and (t.dtype != dt or not t.is_contiguous() or t.numel() != n * self.top_k or t.device != dst.device):
                raise ValueError("ids (int32) and weights (float32) must be contiguous [tokens, top_k] tensors on the layer's device")
        dev = _device_of(dst, x, self._keep[0])
        size = self.workspace_bytes(n)
        if stream is None:
            space = torch.empty(size, dtype=torch.uint8, device=dst.device)
        else:
            # torch takes the handle 0, the default stream's, for none at all and makes a stream of its own
            owner = torch.cuda.ExternalStream(stream, device=dst.device) if stream else torch.cuda.default_stream(dst.device)
            with torch.cuda.stream(owner):
                space = torch.empty(size, dtype=torch.uint8, device=dst.device)
        _call(dev, stream, lib.ggq_moe_device, self._ref, _elem(x), x.data_ptr(), xs, n, _elem(dst), dst.data_ptr(), ys,
              ids.data_ptr() if ids is not None else None, weights.data_ptr() if weights is not None else None, space.data_ptr(), size)
