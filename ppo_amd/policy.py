"""Policies whose actions are tokens: the rules that shape their logits, neglogp and entropy of an action, and the clipped
objective over a gathered minibatch with its gradient.  The reference computes these inside its learner for a handful of
actions (ppo/src/model/learner.rs:112-244, ppo/src/model/util.rs:3-33); the semantics of each call are in include/ppo_xp.h.

Everything runs on torch's current stream of the logits' device, allocates its results with torch and never synchronises, so
the calls may be captured into a HIP graph.  Gradients are returned, not recorded: `logits.backward(r.dlogits)` hands them on.
Wrong arguments raise PpoXpPanic before anything is launched.
"""
from __future__ import annotations

import struct
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import EINVAL, PpoXpPanic, check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_RULES = struct.Struct("19q4f2i")                 # ppo_xp_logit_rules
_BATCH = struct.Struct("6Q")                      # ppo_xp_policy_batch
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda d: torch.cuda.current_stream(d).cuda_stream)


def _panic(msg):
    raise PpoXpPanic(EINVAL, msg)


def _matrix(t, what):
    """(rows, columns, stride of a row) of a 2-d CUDA tensor of a supported type whose rows are contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 2 or t.dtype not in _DTYPES:
        _panic(f"{what}: a 2-d CUDA tensor of f32, bf16 or f16 expected")
    (rows, cols), (sr, sc) = t.shape, t.stride()
    if (sc != 1 and cols > 1) or (sr < cols and rows > 1):
        _panic(f"{what}: rows must be contiguous and must not overlap")
    return rows, cols, max(sr, cols)


def _vector(t, n, dtype, d, what):
    """Address of a contiguous vector of n elements on GPU `d`."""
    try:
        if t.dtype is dtype and t.get_device() == d and t.dim() == 1 and t.numel() == n and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _panic(f"{what}: contiguous {dtype} tensor of {n} on cuda:{d} expected")


def _like(t, out, what):
    """`out`, or a new tensor of t's shape and type; and the stride of its rows."""
    if out is None:
        return torch.empty(t.shape, dtype=t.dtype, device=t.device), t.shape[1]
    if not isinstance(out, torch.Tensor) or out.dtype is not t.dtype or out.device != t.device or out.shape != t.shape:
        _panic(f"{what}: out must have the logits' shape, type and device")
    return out, _matrix(out, what)[2]


def _row_value(v, rows, d, what):
    """(pointer, scalar) of a rule given as one number or as one f32 per row."""
    if isinstance(v, torch.Tensor):
        return _vector(v, rows, torch.float32, d, what), 1.0
    return 0, float(v)


def _rules(t, rows, vocab, history, hist_row, hist_begin, gen_begin, hist_end, repetition, presence, frequency, bias, mask, mask_row,
           temperature):
    d, i32 = t.get_device(), torch.int32
    hp = hsr = hst = hrows = hlen = 0
    bits = 64
    ip = [0, 0, 0, 0]
    if history is not None:
        if not isinstance(history, torch.Tensor) or history.get_device() != d or history.dim() != 2 or history.dtype not in (torch.int64, i32):
            _panic("history: a 2-d int64 or int32 tensor [rows, positions] on the logits' device expected")
        hp, (hrows, hlen), (hsr, hst) = history.data_ptr(), history.shape, history.stride()
        bits = 64 if history.dtype is torch.int64 else 32
        if hist_row is None and hrows != rows:
            _panic(f"history: {hrows} rows for {rows} rows of logits (pass hist_row)")
        for k, (v, name) in enumerate(((hist_row, "hist_row"), (hist_begin, "hist_begin"), (gen_begin, "gen_begin"), (hist_end, "hist_end"))):
            if v is not None:
                ip[k] = _vector(v, rows, i32, d, name)
    elif not (hist_row is hist_begin is gen_begin is hist_end is None):
        _panic("hist_row, hist_begin, gen_begin and hist_end belong to a history")
    rp, rep = _row_value(repetition, rows, d, "repetition")
    pp, pres = _row_value(presence, rows, d, "presence")
    fp, freq = _row_value(frequency, rows, d, "frequency")
    tp, temp = _row_value(temperature, rows, d, "temperature")
    bp = bs = 0
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.get_device() != d or bias.dtype is not torch.float32 or bias.shape not in ((vocab,), (rows, vocab)) or \
                (vocab > 1 and bias.stride(-1) != 1):
            _panic("bias: f32 tensor [vocab] or [rows, vocab] with contiguous rows on the logits' device expected")
        bp, bs = bias.data_ptr(), (bias.stride(0) if bias.dim() == 2 and rows > 1 else 0)
    mp = ms = mrows = mrp = kind = 0
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.get_device() != d or mask.dim() not in (1, 2):
            _panic("mask: a tensor [rows, ...] or [...] on the logits' device expected")
        if mask.dtype in (torch.bool, torch.uint8):
            kind, need = 2, vocab
        elif mask.dtype in (torch.int32, torch.uint32):
            kind, need = 1, (vocab + 31) // 32
        else:
            _panic("mask: bool / uint8 per token, or int32 words of 32 tokens expected")
        mrows = mask.shape[0] if mask.dim() == 2 else 1
        if mask.shape[-1] != need or (need > 1 and mask.stride(-1) != 1):
            _panic(f"mask: contiguous rows of {need} expected")
        if mask_row is not None:
            mrp = _vector(mask_row, rows, i32, d, "mask_row")
        elif mask.dim() == 2 and mrows != rows:
            _panic(f"mask: {mrows} rows for {rows} rows of logits (pass mask_row)")
        mp, ms = mask.data_ptr(), (mask.stride(0) if mask.dim() == 2 and mrows > 1 else 0)
        if mrows == 0:
            kind = 0
    elif mask_row is not None:
        _panic("mask_row belongs to a mask")
    return _RULES.pack(hp, hsr, hst, hrows, hlen, *ip, rp, pp, fp, tp, bp, bs, mp, ms, mrows, mrp, rep, pres, freq, temp, bits, kind)


def shape_logits(logits, *, history=None, hist_row=None, hist_begin=None, gen_begin=None, hist_end=None, repetition=1.0, presence=0.0,
                 frequency=0.0, bias=None, mask=None, mask_row=None, temperature=1.0, out=None):
    """Logits [rows, vocab] under the rules an action is drawn with (ppo_xp_shape_logits).

    history [H, L] int64 / int32 token ids of any strides - a buffer's actions column is
    `buffer.stream_view("actions").view(T, N).t()` - read at [hist_begin, hist_end) of row hist_row[r] (default: row r, all of it);
    tokens from gen_begin on count for frequency and presence.  repetition, presence, frequency, temperature: a number or one f32
    per row.  bias f32 [vocab] or [rows, vocab].  mask: bool / uint8 [.., vocab] or int32 words [.., ceil(vocab / 32)], set = allowed,
    one row for all, one per row, or picked by mask_row (a negative one leaves its row free).  `out` may be `logits`."""
    rows, vocab, stride = _matrix(logits, "shape_logits")
    rules = _rules(logits, rows, vocab, history, hist_row, hist_begin, gen_begin, hist_end, repetition, presence, frequency, bias, mask,
                   mask_row, temperature)
    out, ostride = _like(logits, out, "shape_logits")
    dev = logits.get_device()
    check(_lib.load().ppo_xp_shape_logits(dev, _raw_stream(dev), _DTYPES[logits.dtype], logits.data_ptr(), stride, out.data_ptr(), ostride,
                                          rows, vocab, rules))
    return out


def shape_logits_backward(grad, logits, *, history=None, hist_row=None, hist_begin=None, hist_end=None, repetition=1.0, mask=None,
                          mask_row=None, temperature=1.0, out=None):
    """d(loss)/d(logits) from grad = d(loss)/d(shape_logits(logits)) (ppo_xp_shape_logits_backward); the rules that have no
    gradient - presence, frequency, bias - are not asked for.  `out` may be `grad`."""
    rows, vocab, stride = _matrix(logits, "shape_logits_backward")
    if not isinstance(grad, torch.Tensor) or grad.dtype is not logits.dtype or grad.device != logits.device or grad.shape != logits.shape:
        _panic("shape_logits_backward: grad must have the logits' shape, type and device")
    gstride = _matrix(grad, "shape_logits_backward")[2]
    rules = _rules(logits, rows, vocab, history, hist_row, hist_begin, None, hist_end, repetition, 0.0, 0.0, None, mask, mask_row, temperature)
    out, ostride = _like(grad, out, "shape_logits_backward")
    dev = logits.get_device()
    check(_lib.load().ppo_xp_shape_logits_backward(dev, _raw_stream(dev), _DTYPES[logits.dtype], grad.data_ptr(), gstride, logits.data_ptr(),
                                                   stride, out.data_ptr(), ostride, rows, vocab, rules))
    return out


def action_stats(logits, actions):
    """(neglogps, entropies) f32 [rows] of int64 `actions` under softmax(logits) (util.rs:3-33): what add_experience_device stores.
    A logit of -inf is a forbidden token, an action of -1 padding (both results 0)."""
    rows, vocab, stride = _matrix(logits, "action_stats")
    L, dt, d = _lib.load(), _DTYPES[logits.dtype], logits.get_device()
    ap = _vector(actions, rows, torch.int64, d, "actions")
    n = L.ppo_xp_policy_workspace(rows, vocab, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=logits.device) if n else None       # a new one each call: see policy_loss
    both = torch.empty(2, rows, dtype=torch.float32, device=logits.device)
    p = both.data_ptr()
    check(L.ppo_xp_action_stats(d, _raw_stream(d), dt, logits.data_ptr(), stride, ap, p, p + 4 * rows, rows, vocab, ws.data_ptr() if n else None, n))
    return both.unbind(0)


@dataclass
class PolicyLoss:
    """What policy_loss gives; all on the device."""
    stats: torch.Tensor       # [6] f32: loss, policy, value, entropy, (nlp - old)^2 / 2, share of clipped rows
    dlogits: torch.Tensor     # [rows, vocab], the logits' type: d(loss)/d(logits)
    dvalues: torch.Tensor     # [rows] f32: d(loss)/d(values)
    neglogps: torch.Tensor    # [rows] f32
    entropies: torch.Tensor   # [rows] f32


def policy_loss(logits, values, batch, *, clip=0.2, ent_coef=0.01, vf_coef=0.5, denom=None, out=None):
    """The clipped objective of an ExperienceBatch and its gradient (learner.rs:165-244; defaults of ModelConfig, config.rs:20-36).

    logits [rows, vocab] and values f32 [rows]: the policy and critic now; `batch` an ExperienceBatch or anything with its actions,
    values, neglogps, returns and advantages.  Rows whose action is -1 are padding: pass the number of real rows as `denom`
    (default: all rows).  `out`: where dlogits go, may be `logits` itself."""
    rows, vocab, stride = _matrix(logits, "policy_loss")
    f32 = torch.float32
    L, dt, d = _lib.load(), _DTYPES[logits.dtype], logits.get_device()
    ptrs = (_vector(batch.actions, rows, torch.int64, d, "batch.actions"), _vector(batch.values, rows, f32, d, "batch.values"),
            _vector(batch.neglogps, rows, f32, d, "batch.neglogps"), _vector(batch.returns, rows, f32, d, "batch.returns"),
            _vector(batch.advantages, rows, f32, d, "batch.advantages"), _vector(values, rows, f32, d, "values"))
    dlogits, dstride = _like(logits, out, "policy_loss")
    # one piece of memory for the workspace and the small results, from torch's allocator: calls on two streams and two captured
    # graphs never share it
    n = -(-L.ppo_xp_policy_workspace(rows, vocab, 1) // 4)
    buf = (torch.empty if rows and vocab else torch.zeros)(n + 3 * rows + 6, dtype=f32, device=logits.device)
    _, dvalues, neglogps, entropies, stats = buf.split((n, rows, rows, rows, 6))
    ws = buf.data_ptr()
    p = ws + 4 * n
    check(L.ppo_xp_policy_loss(d, _raw_stream(d), dt, logits.data_ptr(), stride, _BATCH.pack(*ptrs), clip, ent_coef, vf_coef,
                               float(rows or 1) if denom is None else float(denom), dlogits.data_ptr(), dstride, p, p + 4 * rows, p + 8 * rows,
                               p + 12 * rows, rows, vocab, ws, 4 * n))
    return PolicyLoss(stats, dlogits, dvalues, neglogps, entropies)
