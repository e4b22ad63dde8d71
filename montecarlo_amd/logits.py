"""Scores, gradients, draws and keys from a language model's logits: the device calls behind a neural password model
(``mc_logits_*`` of include/mi355mc.h), next to what ``montecarlo_amd.engine`` does for the compiled tables.

The caller's model gives a row of logits over V tokens for every place; all results are in the units of the Monte Carlo path
(-log2 p; keys as float64), so ``logits_keys`` feeds ``MonteCarloLib`` directly.  Tensors live on one GPU; every call runs
on torch's current stream of that GPU, waits for nothing and may be captured into a graph.  No value of -log2 p, entropy or key
is below 0.  The last bits of sums in 32 bits depend on how a launch deals a row to lanes, which goes by the number of rows and
of tokens: the same row scored in calls of other sizes, or scored and drawn from, may differ there.  No CPU fallback: tensors
that are not on a GPU are refused."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as nv

OUTSIDE, SKIP = -1, -2     # token ids: not in the model (impossible); not to be looked at (padding, an ended sample)
MAX_TOP = 64
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class LogitScores(NamedTuple):
    ml2p: torch.Tensor                            # float32, -log2 p of the given tokens
    entropy: Optional[torch.Tensor] = None        # float32, bits
    top_tokens: Optional[torch.Tensor] = None     # int32 [..., top]
    top_ml2p: Optional[torch.Tensor] = None       # float32 [..., top]


class LogitGradient(NamedTuple):
    ml2p: torch.Tensor
    entropy: Optional[torch.Tensor]
    grad: torch.Tensor                            # the logits' shape and type, contiguous


class LogitDraws(NamedTuple):
    tokens: torch.Tensor                          # int32
    ml2p: torch.Tensor                            # float32


def _rows(logits: torch.Tensor, most: int = 3):
    """(dtype code, outer, inner, vocab, outer stride, inner stride, shape of the rows) of logits [V], [N, V] or [B, L, V]."""
    if not logits.is_cuda:
        raise ValueError("logits: a tensor on the GPU is needed (there is no CPU fallback)")
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits: float32, float16 or bfloat16, not {logits.dtype}")
    shape, strides = tuple(logits.shape), logits.stride()
    dims = len(shape)
    if not 1 <= dims <= most:
        raise ValueError(f"logits: 1 to {most} dimensions, the last one over the tokens; got {shape}")
    vocab = shape[-1]
    if vocab == 0:
        raise ValueError("logits: no tokens")
    if strides[-1] != 1 and vocab > 1:
        raise ValueError("logits: the tokens of a row must be adjacent (stride 1 in the last dimension)")
    if dims == 3:
        return code, shape[0], shape[1], vocab, strides[0], strides[1], shape[:2]
    if dims == 2:
        return code, 1, shape[0], vocab, 0, strides[0], shape[:1]
    return code, 1, 1, vocab, 0, 0, ()


def _beside(name: str, t: torch.Tensor, dev: torch.device, rows: tuple, dtypes):
    """Strides (outer, inner) of a tensor with one value for every row."""
    if t.device != dev:
        raise ValueError(f"{name}: on {t.device}, the logits are on {dev}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.shape != rows:
        raise ValueError(f"{name}: shape {tuple(t.shape)} for rows {rows}")
    s = t.stride()
    return s if len(s) == 2 else (0, s[0]) if s else (0, 0)


def _temperature(t) -> float:
    t = float(t)
    if not 1e-30 <= t <= 1e30:
        raise ValueError(f"temperature: a positive number (1e-30 .. 1e30), not {t}")
    return t


def _call(device: torch.device, fn, *args):
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        nv.check(rc)


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    """A call's own, held until its launches are queued; then its memory goes back to torch's pool of the current stream."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


_INTS, _F32, _F64, _BOOL = (torch.int64, torch.int32), (torch.float32,), (torch.float64,), (torch.bool,)


def logits_score(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, entropy: bool = False,
                 top: int = 0) -> LogitScores:
    """-log2 p of ``tokens`` (int32 or int64, one for every row of ``logits``) under softmax(logits / temperature), with the
    rows' entropy in bits and the ``top`` (at most 64) most probable tokens where asked for, in one reading of the logits.

    Any strides are taken as they are (``logits[:, :-1]`` beside ``tokens[:, 1:]`` costs no copy).  ``SKIP`` marks
    rows that are not to be read; any other id outside the vocabulary scores +inf, as does a token whose logit is -inf.
    Alternatives are in the order of the logits, equal ones by the lower id; where fewer than ``top`` have any
    probability the rest is ``OUTSIDE`` with +inf."""
    code, outer, inner, vocab, os, is_, rows = _rows(logits)
    dev = logits.device
    tos, tis = _beside("tokens", tokens, dev, rows, _INTS)
    temperature = _temperature(temperature)
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top: 0 .. {min(MAX_TOP, vocab)} alternatives, not {top}")
    ml2p = logits.new_empty(rows, dtype=torch.float32)
    ent = logits.new_empty(rows, dtype=torch.float32) if entropy else None
    ids = logits.new_empty(rows + (top,), dtype=torch.int32) if top else None
    vals = logits.new_empty(rows + (top,), dtype=torch.float32) if top else None
    need = nv.lib.mc_logits_score_workspace_bytes(code, outer * inner, vocab, top) if vocab > 2048 else 0
    ws = _workspace(need, dev)
    _call(dev, nv.lib.mc_logits_score, logits.data_ptr(), code, outer, inner, vocab, os, is_, tokens.data_ptr(),
          tokens.element_size(), tos, tis, temperature, ml2p.data_ptr(), _ptr(ent), top, _ptr(ids), _ptr(vals),
          _ptr(ws), need)
    return LogitScores(ml2p, ent, ids, vals)


def logits_gradient(logits: torch.Tensor, tokens: torch.Tensor, weights: torch.Tensor, *,
                    entropy_weights: Optional[torch.Tensor] = None, temperature: float = 1.0,
                    out: Optional[torch.Tensor] = None) -> LogitGradient:
    """The gradient for ``logits`` of sum(weights * ml2p) + sum(entropy_weights * entropy), with ml2p and (where
    ``entropy_weights`` is given) entropy as ``logits_score`` returns them.  ``weights``: float32, one for every row; a training
    program passes what its loss multiplies each token's -log2 p with (ln 2 / tokens for a mean in nats) and hands the
    result to ``logits.backward(grad)``.  Skipped rows and rows with no token left have gradient 0; a token outside
    the model contributes none.  ``out``: where to put it -- contiguous, of the logits' shape and type, either the
    logits themselves (overwritten) or memory apart from everything that goes in."""
    code, outer, inner, vocab, os, is_, rows = _rows(logits)
    dev = logits.device
    tos, tis = _beside("tokens", tokens, dev, rows, _INTS)
    wos, wis = _beside("weights", weights, dev, rows, _F32)
    eos, eis = _beside("entropy_weights", entropy_weights, dev, rows, _F32) if entropy_weights is not None else (0, 0)
    temperature = _temperature(temperature)
    if out is None:
        grad = logits.new_empty(logits.shape)
    else:
        grad = out
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or not out.is_contiguous():
            raise ValueError("out: a contiguous tensor of the logits' shape, type and device is needed")
        lo, hi = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
        for name, t in (("logits", logits), ("tokens", tokens), ("weights", weights), ("entropy_weights", entropy_weights)):
            if t is None or t.numel() == 0 or (t is out or (name == "logits" and t.data_ptr() == lo and t.is_contiguous())):
                continue
            first = t.data_ptr()
            last = first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
            if first < hi and lo < last:
                raise ValueError(f"out overlaps {name}")
    ml2p = logits.new_empty(rows, dtype=torch.float32)
    ent = logits.new_empty(rows, dtype=torch.float32) if entropy_weights is not None else None
    need = nv.lib.mc_logits_gradient_workspace_bytes(code, outer * inner, vocab) if vocab > 2048 else 0
    ws = _workspace(need, dev)
    _call(dev, nv.lib.mc_logits_gradient, logits.data_ptr(), code, outer, inner, vocab, os, is_, tokens.data_ptr(),
          tokens.element_size(), tos, tis, temperature, weights.data_ptr(), wos, wis, _ptr(entropy_weights), eos, eis,
          ml2p.data_ptr(), _ptr(ent), grad.data_ptr(), _ptr(ws), need)
    if out is not None:
        torch.autograd.graph.increment_version(out)  # (what autograd saved of it is gone: its backward must notice)
    return LogitGradient(ml2p, ent, grad)


def logits_draw(logits: torch.Tensor, uniforms: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
                live: Optional[torch.Tensor] = None, seed: Optional[int] = None, first_id: int = 0,
                draw: int = 0) -> LogitDraws:
    """One token from every row of ``logits`` ([V] or [N, V]) by inversion, with the -log2 p it was drawn with: the first token
    whose running sum of probabilities exceeds the row's uniform, decided as sums in 64 bits decide it.

    ``uniforms``: float64 in [0, 1), one a row (injected, as ``DeviceModel.sample_injected``); without them row r takes the uniform
    (``seed``, ``first_id`` + r, ``draw``) of the stream that ``DeviceModel.sample`` draws from, so a batch may be cut
    anywhere (what is captured into a graph keeps its seed and draw: replays that are to draw anew take ``uniforms``).  A row's token
    comes with one value, whatever its uniform.  ``live``: bool, rows that are False are not read (``SKIP``, 0).  A row with no
    token left gives ``OUTSIDE`` and +inf."""
    code, _, rows, vocab, _, stride, shape = _rows(logits, 2)
    temperature = _temperature(temperature)
    dev = logits.device
    if (uniforms is None) == (seed is None):
        raise ValueError("either uniforms or a seed is needed")
    if uniforms is not None:
        _beside("uniforms", uniforms, dev, shape, _F64)
        uniforms = uniforms.contiguous()
    if live is not None:
        _beside("live", live, dev, shape, _BOOL)
        live = live.contiguous()
    tokens = logits.new_empty(shape, dtype=torch.int32)
    ml2p = logits.new_empty(shape, dtype=torch.float32)
    need = nv.lib.mc_logits_draw_workspace_bytes(code, rows, vocab) if vocab > 2048 else 0
    ws = _workspace(need, dev)
    _call(dev, nv.lib.mc_logits_draw, logits.data_ptr(), code, rows, vocab, stride, temperature, _ptr(uniforms),
          (seed or 0) & 0xFFFFFFFFFFFFFFFF, first_id & 0xFFFFFFFFFFFFFFFF, draw & 0xFFFFFFFF, _ptr(live), tokens.data_ptr(),
          ml2p.data_ptr(), _ptr(ws), need)
    return LogitDraws(tokens, ml2p)


def logits_keys(ml2p: torch.Tensor, lengths: Optional[torch.Tensor] = None, *,
                offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """-log2 p of whole passwords as float64 keys (what ``MonteCarloLib`` takes): the sums in 64 bits of their tokens'.
    Padded: ``ml2p`` [B, L] with ``lengths`` [B] (int32 or int64; None: L each).  Packed: ``ml2p`` [N] with ``offsets``
    [B + 1] (int64, ascending).  A password with an impossible token is 1022.0, as everywhere in this package, and no key is
    below 0, whatever roundings the values hold: the rank indexes sort the bits of non-negative numbers."""
    if not ml2p.is_cuda:
        raise ValueError("ml2p: a tensor on the GPU is needed (there is no CPU fallback)")
    if ml2p.dtype != torch.float32:
        raise TypeError(f"ml2p: float32, not {ml2p.dtype}")
    dev = ml2p.device
    for name, t, dtypes in (("lengths", lengths, _INTS), ("offsets", offsets, (torch.int64,))):
        if t is not None:
            if t.device != dev:
                raise ValueError(f"{name}: on {t.device}, ml2p is on {dev}")
            if t.dtype not in dtypes or t.dim() != 1:
                raise TypeError(f"{name}: one dimension of {' or '.join(str(d) for d in dtypes)}")
    if offsets is not None:
        if lengths is not None:
            raise ValueError("offsets or lengths, not both")
        if ml2p.dim() != 1 or offsets.numel() == 0:
            raise ValueError("packed: ml2p of one dimension and at least one offset")
        ml2p, offsets = ml2p.contiguous(), offsets.contiguous()
        count, stride, longest = offsets.numel() - 1, 0, ml2p.numel()
    else:
        if ml2p.dim() != 2 or (lengths is not None and lengths.numel() != ml2p.shape[0]):
            raise ValueError("padded: ml2p [B, L] and lengths [B]")
        if ml2p.stride(1) != 1 and ml2p.shape[1] > 1:
            ml2p = ml2p.contiguous()
        lengths = lengths.contiguous() if lengths is not None else None
        count, stride, longest = ml2p.shape[0], ml2p.stride(0), ml2p.shape[1]
    keys = ml2p.new_empty(count, dtype=torch.float64)
    _call(dev, nv.lib.mc_logits_keys, ml2p.data_ptr(), _ptr(offsets), _ptr(lengths),
          lengths.element_size() if lengths is not None else 0, count, stride, longest, keys.data_ptr())
    return keys
