"""Policies whose actions are tokens: the rules that shape their logits, neglogp and entropy of an action, and the clipped
objective over a gathered minibatch with its gradient.  The reference computes these inside its learner for a handful of
actions (ppo/src/model/learner.rs:112-244, ppo/src/model/util.rs:3-33); the semantics of each call are in include/ppo_xp.h.

Everything runs on torch's current stream of the logits' device, allocates its results with torch and never synchronises, so
the calls may be captured into a HIP graph.  Gradients are returned, not recorded: `logits.backward(r.dlogits)` hands them on.
Wrong arguments raise PpoXpPanic before anything is launched.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

_call = _lib.bound                                # csrc/torchcall.cpp: arguments checked, results allocated, launched


def shape_logits(logits, *, history=None, hist_row=None, hist_begin=None, gen_begin=None, hist_end=None, repetition=1.0, presence=0.0,
                 frequency=0.0, bias=None, mask=None, mask_row=None, temperature=1.0, out=None):
    """Logits [rows, vocab] under the rules an action is drawn with (ppo_xp_shape_logits).

    history [H, L] int64 / int32 token ids of any strides - a buffer's actions column is
    `buffer.stream_view("actions").view(T, N).t()` - read at [hist_begin, hist_end) of row hist_row[r] (default: row r, all of it);
    tokens from gen_begin on count for frequency and presence.  repetition, presence, frequency, temperature: a number or one f32
    per row; repetition and temperature at least 2^-126 (a number below is refused, a row's own counts as 2^-126).  bias f32 [vocab] or [rows, vocab].  mask: bool / uint8 [.., vocab] or int32 words [.., ceil(vocab / 32)], set = allowed,
    one row for all, one per row, or picked by mask_row (a negative one leaves its row free).  `out` may be `logits`."""
    return _call.shape(logits, history, hist_row, hist_begin, gen_begin, hist_end, repetition, presence, frequency, bias, mask, mask_row,
                       temperature, out)


def shape_logits_backward(grad, logits, *, history=None, hist_row=None, hist_begin=None, hist_end=None, repetition=1.0, mask=None,
                          mask_row=None, temperature=1.0, out=None):
    """d(loss)/d(logits) from grad = d(loss)/d(shape_logits(logits)) (ppo_xp_shape_logits_backward); the rules that have no
    gradient - presence, frequency, bias - are not asked for.  `out` may be `grad`."""
    return _call.shape_backward(grad, logits, history, hist_row, hist_begin, None, hist_end, repetition, 0.0, 0.0, None, mask, mask_row,
                                temperature, out)


def action_stats(logits, actions):
    """(neglogps, entropies) f32 [rows] of int64 `actions` under softmax(logits) (util.rs:3-33): what add_experience_device stores.
    A logit of -inf is a forbidden token, an action of -1 padding (both results 0)."""
    return _call.stats(logits, actions)


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
    (default: all rows); rows / S for gradients and statistics S times as large, which f16 gradients need (elements below 2^-25 become
    0).  `out`: where dlogits go, may be `logits` itself."""
    return PolicyLoss(*_call.loss(logits, values, batch, clip, ent_coef, vf_coef, denom, out))
