"""The token-policy operators refuse wrong arguments before anything is launched: through the C ABI with addresses that are never
read, and through the Python calls.  Runs without a GPU."""
import struct

import pytest
import torch

import ppo_amd
from ppo_amd import _lib

L = _lib.load()
RULES = struct.Struct("19q4f2i")                  # ppo_xp_logit_rules
P = 0x10000            # an address nothing looks at: every call below is refused first


def rules(**kw):
    d = dict(history=0, hist_row_stride=0, hist_tok_stride=0, hist_rows=0, hist_len=0, hist_row=0, hist_begin=0, gen_begin=0, hist_end=0,
             repetition_rows=0, presence_rows=0, frequency_rows=0, temperature_rows=0, bias=0, bias_stride=0, mask=0, mask_stride=0,
             mask_rows=0, mask_row=0, repetition=1.0, presence=0.0, frequency=0.0, temperature=1.0, history_bits=64, mask_kind=0)
    assert set(kw) <= set(d)
    d.update(kw)
    return RULES.pack(*d.values())


def shape(dtype=0, logits=P, ls=100, out=P, os_=100, rows=4, vocab=100, r=None):
    return L.ppo_xp_shape_logits(0, None, dtype, logits, ls, out, os_, rows, vocab, rules() if r is None else r)


def refused(rc, text):
    assert rc == _lib.EINVAL and text in _lib.last_error(), (rc, _lib.last_error())


def test_shape_refusals():
    refused(shape(dtype=3), "unknown element type")
    refused(shape(logits=None), "NULL")
    refused(shape(out=None), "NULL")
    refused(shape(ls=99), "lie 99 apart")
    refused(shape(os_=0), "lie 0 apart")
    refused(shape(vocab=(1 << 30) + 1, ls=1 << 31, os_=1 << 31), "2^30")
    refused(L.ppo_xp_shape_logits(0, None, 0, P, 100, P, 100, 4, 100, None), "rules is NULL")
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        refused(shape(r=rules(repetition=bad)), "repetition")
        refused(shape(r=rules(temperature=bad)), "temperature")
    for bad in (float("inf"), float("nan")):
        refused(shape(r=rules(presence=bad)), "presence")
        refused(shape(r=rules(frequency=bad)), "frequency")
    h = dict(history=P, hist_row_stride=8, hist_tok_stride=1, hist_rows=4, hist_len=8)
    refused(shape(r=rules(**{**h, "history_bits": 16})), "16-bit")
    refused(shape(r=rules(**{**h, "hist_rows": 3})), "3 history rows for 4")
    refused(shape(r=rules(**{**h, "hist_len": -1})), "history shape")
    refused(shape(r=rules(**{**h, "hist_tok_stride": -1})), "history shape")
    refused(shape(r=rules(bias=P, bias_stride=99)), "bias")
    refused(shape(r=rules(mask_kind=3, mask=P, mask_rows=4, mask_stride=100)), "mask kind")
    refused(shape(r=rules(mask_kind=1, mask_rows=4, mask_stride=4)), "mask is NULL")
    refused(shape(r=rules(mask_kind=1, mask=P, mask_rows=4, mask_stride=3)), "stride of 3")
    refused(shape(r=rules(mask_kind=2, mask=P, mask_rows=3, mask_stride=100)), "3 mask rows for 4")
    refused(shape(rows=1 << 31, vocab=100), "too many")
    assert shape(rows=0) == 0 and shape(vocab=0) == 0


def test_backward_refusals():
    f = lambda g=P, gs=100, l=P, ls=100, o=P, os_=100: L.ppo_xp_shape_logits_backward(0, None, 0, g, gs, l, ls, o, os_, 4, 100, rules())  # noqa: E731
    refused(f(g=None), "NULL")
    refused(f(l=None), "NULL")
    refused(f(o=None), "NULL")
    refused(f(gs=10), "apart")
    refused(f(ls=10), "apart")
    refused(f(os_=10), "apart")


def test_stats_and_loss_refusals():
    need = L.ppo_xp_policy_workspace(4, 1 << 20, 0)
    st = lambda dtype=0, a=P, n=P, e=P, rows=4, ws=P, nb=1 << 40: \
        L.ppo_xp_action_stats(0, None, dtype, P, 1 << 20, a, n, e, rows, 1 << 20, ws, nb)  # noqa: E731
    refused(st(dtype=-1), "element type")
    refused(st(a=None), "NULL")
    refused(st(n=None), "NULL")
    refused(st(e=None), "NULL")
    refused(st(rows=1 << 31), "too many")
    assert need > 0                                        # few rows of a million tokens are split over workgroups
    refused(st(ws=None), "workspace")
    refused(st(nb=need - 1), "workspace")
    refused(st(ws=P + 8), "workspace")
    assert L.ppo_xp_policy_workspace(4, 100, 0) == 0 and L.ppo_xp_policy_workspace(0, 100, 1) == 0
    assert st(rows=0) == 0

    def loss(batch=(P,) * 6, clip=0.2, ent=0.01, vf=0.5, denom=4.0, d=P, ds=100, dv=P, stats=P, ws=P, nb=1 << 40):
        b = struct.pack("6Q", *batch) if batch else None
        return L.ppo_xp_policy_loss(0, None, 0, P, 100, b, clip, ent, vf, denom, d, ds, dv, P, P, stats, 4, 100, ws, nb)
    refused(loss(batch=None), "NULL")
    for k in range(6):
        refused(loss(batch=tuple(0 if i == k else P for i in range(6))), "NULL")
    for kw in (dict(clip=-0.1), dict(clip=float("nan")), dict(ent=float("inf")), dict(vf=float("nan"))):
        refused(loss(**kw), "finite")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        refused(loss(denom=bad), "denom")
    refused(loss(d=None), "NULL")
    refused(loss(ds=10), "apart")
    refused(loss(dv=None), "NULL")
    refused(loss(stats=None), "NULL")
    need = L.ppo_xp_policy_workspace(4, 100, 1)
    assert need > 0
    refused(loss(ws=None), "workspace")
    refused(loss(nb=need - 1), "workspace")
    refused(loss(ws=P + 4), "workspace")


def test_row_store_refusals():
    q = lambda dtype=0, rows=P, rs=64, n=4, w=64, f=1, g=64, c=P, cs=64, s=P, ss=1, store=8, at=0: \
        L.ppo_xp_quantize_rows(0, None, dtype, rows, rs, n, w, f, g, c, cs, s, ss, store, at)  # noqa: E731
    refused(q(dtype=7), "element type")
    refused(q(f=0), "format")
    refused(q(g=48), "group 48")
    refused(q(g=8), "group 8")
    refused(q(w=0), "width 0")
    refused(q(c=None), "NULL")
    refused(q(s=None), "NULL")
    refused(q(cs=63), "do not fit")
    refused(q(w=65, cs=65, rs=65), "do not fit")
    refused(q(rows=None), "NULL")
    refused(q(rs=63), "apart")
    refused(q(at=5), "rows 5 .. 9 of a store of 8")
    refused(q(at=2**64 - 2), "of a store of 8")
    assert q(n=0) == 0
    d = lambda dtype=0, c=P, cs=64, s=P, ss=1, store=8, w=64, f=1, g=64, idx=P, bits=32, at=0, n=4, o=P, os_=64: \
        L.ppo_xp_dequantize_rows(0, None, dtype, c, cs, s, ss, store, w, f, g, idx, bits, at, n, o, os_)  # noqa: E731
    refused(d(bits=16), "16 bits")
    refused(d(store=0), "empty store")
    refused(d(o=None), "NULL")
    refused(d(os_=63), "do not fit")
    refused(d(idx=None, at=6), "rows 6 .. 10")
    refused(d(f=4), "format")
    assert d(n=0) == 0


def test_no_gpu_fails_loudly():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert shape() == _lib.ENODEV
    assert L.ppo_xp_quantize_rows(0, None, 0, P, 64, 4, 64, 1, 64, P, 64, P, 1, 8, 0) == _lib.ENODEV


def test_python_refusals():
    x = torch.zeros(2, 8)
    for call in (lambda: ppo_amd.shape_logits(x), lambda: ppo_amd.shape_logits_backward(x, x),
                 lambda: ppo_amd.action_stats(x, torch.zeros(2, dtype=torch.int64)),
                 lambda: ppo_amd.policy_loss(x, torch.zeros(2), None),
                 lambda: ppo_amd.QuantizedRows(4, 8, format="int5"), lambda: ppo_amd.QuantizedRows(4, 0),
                 lambda: ppo_amd.QuantizedRows.of(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1), 8, "int8", 64)):
        with pytest.raises(ppo_amd.PpoXpPanic) as e:
            call()
        assert e.value.code == _lib.EINVAL
