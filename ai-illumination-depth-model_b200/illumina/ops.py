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
allocated too. Inputs must stay alive until the work is done. Autograd is not
part of them: a tensor that requires a gradient is refused (unless under
torch.no_grad()), and so is one with a forward-mode tangent; the backward
passes are calls of their own. Errors are IlluminaError with status
INVALID_ARG.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

from ._lib import ACT, ENGINE, INVALID_ARG, IlluminaError, check, lib, ptr, stream_handle


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


def _load():
    """The torch binding (built beside the library): it checks the tensors and allocates the results."""
    global _native
    import torch  # noqa: F401 - the binding's libraries
    lib()
    from . import _torch_ops
    _native = _torch_ops
    return _native


_native = None


class _On:
    """Makes a device and a stream (a torch stream, a handle, or None for the device's current one) current for a scope;
    the scope's value is the cudaStream_t."""

    def __init__(self, device, stream):
        import torch
        _require(device.type == "cuda", "the tensors of a call must be CUDA tensors")
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=device)
        # a stream of another device would leave the call on the current stream of this one
        _require(stream is None or stream.device == device, f"stream must be a stream of {device}")
        self._scopes = [torch.cuda.device(device)] + ([] if stream is None else [torch.cuda.stream(stream)])
        self._handle = (torch.cuda.current_stream(device) if stream is None else stream).cuda_stream

    def __enter__(self):
        for s in self._scopes:
            s.__enter__()
        return self._handle

    def __exit__(self, *exc):
        for s in reversed(self._scopes):
            s.__exit__(*exc)


def _call(name, stream, first, *args):
    """A native call on the stream given, or on the current one of the first tensor's device."""
    call = getattr(_native or _load(), name)
    if stream is None:
        return call(first, *args)
    with _On(first.device, stream):
        return call(first, *args)


def layerNorm(x, weight=None, bias=None, eps=1e-6, out=None, stream=None):
    """Layer norm over the last dimension: (y, mean, rstd), the float32 statistics [rows] being what layerNormBackward
    needs. weight, bias: float32 [width] or None. out may be x."""
    return _call("layer_norm", stream, x, weight, bias, eps, out)


def layerNormBackward(dy, x, mean, rstd, weight=None, needWeight=True, stream=None):
    """Gradients of layerNorm: (dx, dw, db); dw and db are float32 [width], None unless needWeight."""
    return _call("layer_norm_backward", stream, dy, x, mean, rstd, weight, needWeight)


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
    both = _call("rotary", stream, q, k, positions, plan.turns, plan.axis, plan.axes, plan.headDim, plan.interleaved,
                 inverse, outQ, outK)
    return both[0] if k is None else both


def attention(q, k, v, scale=None, causalBlock=0, qLens=None, kLens=None, stream=None):
    """softmax(scale q k') v: (out [batch, tokens, heads, headDim], lse float32 [batch, heads, tokens]).

    q [batch, queries, heads, headDim]; k, v [batch, keys, keyHeads, headDim], heads a multiple of keyHeads, headDim at
    most 128; scale defaults to headDim**-0.5. qLens, kLens (int32 [batch]): lengths of a padded batch; padding may
    hold anything and its rows come back as zeros. causalBlock n: the last query stands at the last key, and a query
    sees its own block of n keys and those before it (1: causal tokens; the tokens of a frame: causal frames). Rows
    that see no key are zeros with lse -inf. In bfloat16 the probabilities are rounded to bfloat16 before their product
    with v (sums, maxima and lse are not): out is about 2.5e-3 of its norm off, where rounding out alone makes 1.7e-3."""
    return _call("attention", stream, q, k, v, scale, causalBlock, qLens, kLens)


def attentionBackward(dOut, q, k, v, out, lse, scale=None, causalBlock=0, qLens=None, kLens=None, stream=None):
    """Gradients (dq, dk, dv) of attention, from its results out and lse and the same masks. In bfloat16 the
    probabilities and their gradients are rounded to bfloat16 before their products, as in attention."""
    return _call("attention_backward", stream, dOut, q, k, v, out, lse, scale, causalBlock, qLens, kLens)


def checkAttention(device=None) -> None:
    """Raises IlluminaError with status TIMEOUT if a tensor-core kernel of an attention call on the device (the current
    one) gave up a bounded wait since this was last reported: the results of that call are undefined. Does not wait for
    the device: ask after the work, a replayed graph's too, has been synchronised. The next attention call on the device
    asks as well, and is not queued when it raises."""
    import torch
    with torch.cuda.device(device):
        check(lib().illumina_op_attention_status())


def setAttentionWaitLimit(cycles: int) -> None:
    """Cycles such a wait may take in the attention calls of this thread from now on; 0 restores the default (about a
    second). Captured calls keep the limit they were captured with."""
    check(lib().illumina_op_attention_set_wait_limit(int(cycles)))
