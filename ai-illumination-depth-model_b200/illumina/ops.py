"""Per-kernel entry points: the analogues of the reference's kernel factories
(makePointwise, makeDepthwisePointwise, makeConv, makeLateral, makeHead,
makePreprocess, makeDepthUpsample under src/model/kernels/). Arguments are
torch CUDA tensors in the reference's logical layouts; each call launches the
same CUDA kernel the model uses.

The token operators at the end (layerNorm, rotary, attention and their
gradients) have no counterpart in the reference: a transformer stage over the
network's feature maps, or over the frames of a clip. They take shaped torch
CUDA tensors of one device, float32 or bfloat16, with any strides over a
contiguous last dimension, and run on `stream` (a torch stream or handle; by
default torch's current stream of that device), where their results are
allocated too. Inputs must stay alive until the work is done. Errors are
IlluminaError with status INVALID_ARG.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
from dataclasses import dataclass

from ._lib import (ACT, ENGINE, INVALID_ARG, PRECISION_BF16, PRECISION_F32, AttentionArgs, IlluminaError, RotaryArgs,
                   check, lib, ptr, stream_handle)

# illumina_rotary_args and illumina_attention_args as one packing each: a call fills some forty fields, and setting
# them one by one takes longer than a small call's kernel
_ROTARY_ARGS = struct.Struct("@iqqiiiiiPPi3q3qPPi3q3qPi3qPP")
_ATTENTION_ARGS = struct.Struct("@iiiiiiiif" + "P3q" * 4 + "PPP" + "P3q" * 4 + "PN")
assert _ROTARY_ARGS.size == C.sizeof(RotaryArgs) and _ATTENTION_ARGS.size == C.sizeof(AttentionArgs)


def set_engine(engine: str) -> None:
    """Engine of this thread's pointwise / dw->pw / lateral entry points: "simt" (default) or "tensor"."""
    check(lib().illumina_set_op_engine(ENGINE[engine]))


def _out(torch, shape, like):
    return torch.empty(shape, dtype=torch.float32, device=like.device)


def pointwise(src, h, w, in_c, weights, bias, out_c, act, residual=None, dst=None, stream=None):
    import torch
    dst = dst if dst is not None else _out(torch, (h * w * out_c,), src)
    check(lib().illumina_op_pointwise(ptr(src), h * w, in_c, ptr(weights), ptr(bias), out_c, ACT[act],
                                      ptr(residual), ptr(dst), stream_handle(stream)))
    return dst


def dwpw(src, in_h, in_w, in_c, dw_w, dw_b, mid_act, pw_w, pw_b, out_c, k, stride, act, residual=None, dst=None,
         stream=None):
    import torch
    pad = (k - 1) >> 1
    oh, ow = (in_h + 2 * pad - k) // stride + 1, (in_w + 2 * pad - k) // stride + 1
    dst = dst if dst is not None else _out(torch, (oh * ow * out_c,), src)
    check(lib().illumina_op_dwpw(ptr(src), in_h, in_w, in_c, ptr(dw_w), ptr(dw_b), ACT[mid_act], ptr(pw_w),
                                 ptr(pw_b), out_c, k, stride, ACT[act], ptr(residual), ptr(dst),
                                 stream_handle(stream)))
    return dst


def conv(src, in_h, in_w, in_c, weights, bias, out_c, k, stride, act, dst=None, stream=None):
    import torch
    pad = (k - 1) >> 1
    oh, ow = (in_h + 2 * pad - k) // stride + 1, (in_w + 2 * pad - k) // stride + 1
    dst = dst if dst is not None else _out(torch, (oh * ow * out_c,), src)
    check(lib().illumina_op_conv(ptr(src), in_h, in_w, in_c, ptr(weights), ptr(bias), out_c, k, stride, ACT[act],
                                 ptr(dst), stream_handle(stream)))
    return dst


def lateral(coarse, ch, cw, skip, skip_c, weights, bias, out_c, act, dst=None, stream=None):
    import torch
    dst = dst if dst is not None else _out(torch, (4 * ch * cw * out_c,), coarse)
    check(lib().illumina_op_lateral(ptr(coarse), ch, cw, ptr(skip), skip_c, ptr(weights), ptr(bias), out_c,
                                    ACT[act], ptr(dst), stream_handle(stream)))
    return dst


def head(src, pixels, in_c, weights, bias, dst=None, stream=None):
    import torch
    dst = dst if dst is not None else _out(torch, (pixels * 4,), src)
    check(lib().illumina_op_head(ptr(src), pixels, in_c, ptr(weights), float(bias), ptr(dst),
                                 stream_handle(stream)))
    return dst


def preprocess(frames, n, layout, size, decode_srgb=True, exposure=1.0, scene=True, stream=None):
    import torch
    inp = _out(torch, (n * size * size * 4,), frames)
    sc = _out(torch, (n * size * size * 4,), frames) if scene else None
    check(lib().illumina_op_preprocess(ptr(frames), n, layout, size, 1 if decode_srgb else 0, float(exposure),
                                       ptr(inp), ptr(sc), stream_handle(stream)))
    return inp, sc


def bilateral(low, lh, lw, low_c, guide, guide_c, range_sigma=0.12, dst=None, stream=None):
    import torch
    dst = dst if dst is not None else _out(torch, (4 * lh * lw,), low)
    check(lib().illumina_op_bilateral(ptr(low), lh, lw, low_c, ptr(guide), guide_c, float(range_sigma), ptr(dst),
                                      stream_handle(stream)))
    return dst


# ---------------------------------------------------------------------------
# Token operators
# ---------------------------------------------------------------------------

def _require(ok, message):
    if not ok:
        raise IlluminaError(INVALID_ARG, message)


class _On:
    """Makes a tensor's device and the call's stream current for a scope; `handle` is the stream's cudaStream_t.
    Usually both are current already: then this is two reads of torch's state."""
    __slots__ = ("handle", "_scopes")

    def __init__(self, torch, device, stream):
        index = device.index
        self._scopes = None
        if stream is None:
            self.handle = torch._C._cuda_getCurrentRawStream(index)
            if torch._C._cuda_getDevice() != index:
                self._scopes = (torch.cuda.device(device),)
        else:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream, device=device)
            self._scopes = (torch.cuda.device(device), torch.cuda.stream(stream))
            self.handle = stream.cuda_stream

    def __enter__(self):
        if self._scopes:
            for s in self._scopes:
                s.__enter__()
        return self.handle

    def __exit__(self, *exc):
        if self._scopes:
            for s in reversed(self._scopes):
                s.__exit__(*exc)


def _precision(torch, name, x):
    if x.dtype == torch.float32:
        return PRECISION_F32
    _require(x.dtype == torch.bfloat16, f"{name} must be float32 or bfloat16")
    return PRECISION_BF16


def _tensor(torch, name, x, like=None, dims=None):
    """Checks a storage tensor: on a CUDA device, contiguous in its last dimension, of `like`'s type and device."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _require(False, f"{name} must be a CUDA tensor")
    shape = x.shape
    if dims is not None and len(shape) != dims:
        _require(False, f"{name} must have {dims} dimensions")
    if not shape or (shape[-1] > 1 and x.stride(-1) != 1):
        _require(False, f"{name} must be contiguous in its last dimension")
    if like is not None and (x.dtype != like.dtype or x.get_device() != like.get_device()):
        _require(False, f"{name} must have the type and device of the others")


def _vector(torch, name, x, n, device, dtype=None):
    """Checks a contiguous vector of n elements (float32 by default) and returns its address; None passes."""
    if x is None:
        return None
    dtype = dtype or torch.float32
    if not (isinstance(x, torch.Tensor) and x.dtype == dtype and x.device == device and x.numel() == n and x.is_contiguous()):
        _require(False, f"{name} must be {n} contiguous {str(dtype)[6:]} values on the device of the others")
    return x.data_ptr()


def _rows(torch, name, x):
    """(rows, width, row stride) of a tensor whose leading dimensions are evenly spaced rows."""
    shape, strides = x.shape, x.stride()
    if len(shape) == 2:
        return shape[0], shape[1], strides[0]
    rows, stride = 1, None
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n != 1:
            if stride is None:
                stride = s
            _require(rows == 0 or s == stride * rows, f"{name} must have evenly spaced rows (reshape it to two dimensions)")
        rows *= n
    return rows, shape[-1], shape[-1] if stride is None else stride


@functools.lru_cache(maxsize=4096)
def _norm_workspace(rows, c):
    size = C.c_size_t(0)
    check(lib().illumina_op_layer_norm_workspace(rows, c, C.byref(size)))
    return size.value


def layerNorm(x, weight=None, bias=None, eps=1e-6, out=None, stream=None):
    """Layer norm over the last dimension: (y, mean, rstd), the float32 statistics [rows] being what layerNormBackward
    needs. weight, bias: float32 [width] or None. out may be x."""
    import torch
    _tensor(torch, "x", x)
    precision = _precision(torch, "x", x)
    rows, c, stride = _rows(torch, "x", x)
    if not c:
        _require(False, "x must not have a width of zero")
    device = x.device
    w = _vector(torch, "weight", weight, c, device)
    b = _vector(torch, "bias", bias, c, device)
    with _On(torch, device, stream) as handle:
        if out is None:
            out, out_stride = x.new_empty(x.shape), c
        else:
            _tensor(torch, "out", out, x)
            _require(out.shape == x.shape, "out must have the shape of x")
            out_stride = _rows(torch, "out", out)[2]
        mean, rstd = torch.empty((2, rows), dtype=torch.float32, device=device).unbind()
        check(lib().illumina_op_layer_norm(precision, x.data_ptr(), stride, rows, c, w, b, eps, out.data_ptr(), out_stride,
                                           mean.data_ptr(), rstd.data_ptr(), handle))
    return out, mean, rstd


def layerNormBackward(dy, x, mean, rstd, weight=None, needWeight=True, stream=None):
    """Gradients of layerNorm: (dx, dw, db); dw and db are float32 [width], None unless needWeight."""
    import torch
    _tensor(torch, "x", x)
    _tensor(torch, "dy", dy, x)
    if dy.shape != x.shape:
        _require(False, "dy must have the shape of x")
    precision = _precision(torch, "x", x)
    rows, c, stride = _rows(torch, "x", x)
    _, _, dy_stride = _rows(torch, "dy", dy)
    if not c:
        _require(False, "x must not have a width of zero")
    device = x.device
    w = _vector(torch, "weight", weight, c, device)
    if mean is None or rstd is None:
        _require(False, "mean and rstd of the forward pass are needed")
    mean_at, rstd_at = _vector(torch, "mean", mean, rows, device), _vector(torch, "rstd", rstd, rows, device)
    with _On(torch, device, stream) as handle:
        dx = x.new_empty(x.shape)
        dw = db = workspace = None
        size = 0
        if needWeight:
            size = _norm_workspace(rows, c)
            dw, db = torch.empty((2, c), dtype=torch.float32, device=device).unbind()
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
        check(lib().illumina_op_layer_norm_backward(precision, dy.data_ptr(), dy_stride, x.data_ptr(), stride, rows, c, w,
                                                    mean_at, rstd_at, dx.data_ptr(), c, ptr(dw), ptr(db), ptr(workspace),
                                                    size, handle))
    return dx, dw, db


@dataclass(frozen=True)
class RotaryPlan:
    """The frequencies of a rotation, made once by createRotary: turns (float64) and axis (int32) of every pair."""
    headDim: int
    axes: int
    interleaved: bool
    turns: object
    axis: object


def createRotary(headDim, sections, base=10000.0, interleaved=False, spectrum="axis", device="cuda"):
    """Rotary positions with len(sections) axes (time, row, column; any number). Axis a has sections[a] consecutive
    pairs. spectrum "axis": its j-th pair turns by position * base**(-j / sections[a]), every axis covers all
    frequencies; "shared": pair i of all P turns by position[axis] * base**(-i / P), the axes share one spectrum.
    Pairs are elements (i, i + P), or neighbours (2i, 2i + 1) when interleaved; elements from 2P on stay."""
    import torch
    sections = [int(n) for n in sections]
    pairs = sum(sections)
    _require(len(sections) > 0 and all(n >= 0 for n in sections), "sections must be counts of pairs")
    _require(pairs >= 1 and 2 * pairs <= headDim, "sections must hold between 1 and headDim / 2 pairs")
    _require(base > 0, "base must be positive")
    _require(spectrum in ("axis", "shared"), 'spectrum must be "axis" or "shared"')
    turns, axis = [], []
    for a, n in enumerate(sections):
        for j in range(n):
            power = j / n if spectrum == "axis" else len(turns) / pairs
            turns.append(base ** -power / (2 * math.pi))
            axis.append(a)
    return RotaryPlan(int(headDim), len(sections), bool(interleaved),
                      torch.tensor(turns, dtype=torch.float64, device=device),
                      torch.tensor(axis, dtype=torch.int32, device=device))


def rotary(q, positions, plan, k=None, inverse=False, outQ=None, outK=None, stream=None):
    """Rotates q [batch, tokens, heads, headDim], and k with its own head count, by positions [axes, tokens] or [axes,
    batch, tokens] (int32 or float32). inverse turns back: the gradient. Returns q's result, or both with k. outQ and
    outK may be q and k."""
    import torch
    _tensor(torch, "q", q, dims=4)
    precision = _precision(torch, "q", q)
    b, t, h, d = q.shape
    _require(d == plan.headDim, f"q must have the plan's {plan.headDim} elements a head")
    _require(plan.turns.device == q.device, "the plan must be on the device of q")
    _require(isinstance(positions, torch.Tensor) and positions.device == q.device and
             positions.dtype in (torch.int32, torch.float32), "positions must be int32 or float32 on the device of q")
    _require(tuple(positions.shape) in ((plan.axes, t), (plan.axes, b, t)),
             "positions must be [axes, tokens] or [axes, batch, tokens]")
    if k is not None:
        _tensor(torch, "k", k, q, 4)
        _require((k.shape[0], k.shape[1], k.shape[3]) == (b, t, d), "k must have the batch, tokens and head size of q")
    ps = positions.stride()
    with _On(torch, q.device, stream) as handle:
        outs, tensors = [], []
        for x, out, name in ((q, outQ, "outQ"), (k, outK, "outK")):
            if x is None:
                tensors += (0, 0, 0, 0, 0, 0, 0, 0, 0)
                continue
            if out is None:
                out = x.new_empty(x.shape)
            else:
                _tensor(torch, name, out, x, 4)
                _require(out.shape == x.shape, f"{name} must have the shape of its input")
            tensors += (x.data_ptr(), out.data_ptr(), x.shape[2], *x.stride()[:3], *out.stride()[:3])
            outs.append(out)
        turns, axis = plan.turns, plan.axis
        args = _ROTARY_ARGS.pack(precision, b, t, d, turns.numel(), plan.axes, plan.interleaved, bool(inverse), *tensors,
                                 positions.data_ptr(), positions.dtype == torch.float32, ps[0],
                                 ps[1] if len(ps) == 3 else 0, ps[-1], turns.data_ptr(), axis.data_ptr())
        check(lib().illumina_op_rotary(args, handle))
    return outs[0] if k is None else tuple(outs)


@functools.lru_cache(maxsize=4096)
def _attention_workspace(precision, b, h, hk, d, tq, tk, backward):
    args = AttentionArgs(precision=precision, batch=b, heads=h, kv_heads=hk, head_dim=d, q_tokens=tq, k_tokens=tk, scale=1.0)
    size = C.c_size_t(0)
    check(lib().illumina_op_attention_workspace(C.byref(args), backward, C.byref(size)))
    return size.value


def _attention(torch, q, k, v, scale, causalBlock, qLens, kLens):
    """Checks an attention call; the leading fields of its arguments, the fields of q, k and v, and the lengths'."""
    _tensor(torch, "q", q, None, 4)
    _tensor(torch, "k", k, q, 4)
    _tensor(torch, "v", v, q, 4)
    (b, tq, h, d), (kb, tk, hk, kd) = q.shape, k.shape
    if k.shape != v.shape or kb != b or kd != d:
        _require(False, "k and v must have q's batch and head size, and one shape")
    if hk < 1 or h % hk:
        _require(False, "q's heads must be a multiple of the key heads")
    _require(1 <= d <= 128, "head sizes from 1 to 128 are supported")
    _require(max(b, h, tq, tk) <= 2 ** 28, "attention: size beyond 2^28")
    _require(isinstance(causalBlock, int) and 0 <= causalBlock < 2 ** 31, "causalBlock must be a token count, 0 for none")
    device = q.device
    lens = (_vector(torch, "qLens", qLens, b, device, torch.int32) or 0,
            _vector(torch, "kLens", kLens, b, device, torch.int32) or 0)
    sizes = (_precision(torch, "q", q), b, h, hk, d, tq, tk)
    return sizes, (causalBlock, d ** -0.5 if scale is None else scale, *_fields(q), *_fields(k), *_fields(v)), lens


def _fields(x):
    return (x.data_ptr(), *x.stride()[:3])


_NO_TENSORS = (0,) * 16


def attention(q, k, v, scale=None, causalBlock=0, qLens=None, kLens=None, stream=None):
    """softmax(scale q k') v: (out [batch, tokens, heads, headDim], lse float32 [batch, heads, tokens]).

    q [batch, queries, heads, headDim]; k, v [batch, keys, keyHeads, headDim], heads a multiple of keyHeads, headDim at
    most 128; scale defaults to headDim**-0.5. qLens, kLens (int32 [batch]): lengths of a padded batch; padding may
    hold anything and its rows come back as zeros. causalBlock n: the last query stands at the last key, and a query
    sees its own block of n keys and those before it (1: causal tokens; the tokens of a frame: causal frames). Rows
    that see no key are zeros with lse -inf."""
    import torch
    sizes, inputs, lens = _attention(torch, q, k, v, scale, causalBlock, qLens, kLens)
    device = q.device
    with _On(torch, device, stream) as handle:
        out = q.new_empty(q.shape)
        lse = torch.empty((sizes[1], sizes[2], sizes[5]), dtype=torch.float32, device=device)
        size = _attention_workspace(*sizes, 0)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        args = _ATTENTION_ARGS.pack(*sizes, *inputs, *_fields(out), *lens, lse.data_ptr(), *_NO_TENSORS,
                                    ptr(workspace) or 0, size)
        check(lib().illumina_op_attention(args, handle))
    return out, lse


def attentionBackward(dOut, q, k, v, out, lse, scale=None, causalBlock=0, qLens=None, kLens=None, stream=None):
    """Gradients (dq, dk, dv) of attention, from its results out and lse and the same masks."""
    import torch
    sizes, inputs, lens = _attention(torch, q, k, v, scale, causalBlock, qLens, kLens)
    for name, x in (("dOut", dOut), ("out", out)):
        _tensor(torch, name, x, q, 4)
        if x.shape != q.shape:
            _require(False, f"{name} must have the shape of q")
    device = q.device
    _require(lse is not None, "lse of the forward pass is needed")
    lse_at = _vector(torch, "lse", lse, sizes[1] * sizes[2] * sizes[5], device)
    with _On(torch, device, stream) as handle:
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        size = _attention_workspace(*sizes, 1)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        args = _ATTENTION_ARGS.pack(*sizes, *inputs, *_fields(out), *lens, lse_at, *_fields(dOut), *_fields(dq),
                                    *_fields(dk), *_fields(dv), workspace.data_ptr(), size)
        check(lib().illumina_op_attention_backward(args, handle))
    return dq, dk, dv
