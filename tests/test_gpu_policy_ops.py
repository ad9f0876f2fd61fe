"""Logit rules, action statistics and the clipped objective against plain 64-bit evaluations of their definitions
(include/ppo_xp.h), at the sizes and masks where they can go wrong.

Tolerances count roundings: u = 2^-24 is half a step of a 32-bit operation, `half(t)` half a step of the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf


def half(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):       # half of the least subnormal: what a rounding near zero can be off by
    return {torch.float64: 0.0, F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}[dtype]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def bits_of(ok):
    """bool [n, V] -> int32 words."""
    n, V = ok.shape
    pad = torch.nn.functional.pad(ok, (0, (-V) % 32)).reshape(n, -1, 32).long()
    w = (pad << torch.arange(32, device="cuda")).sum(2)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


# ---- rules ----------------------------------------------------------------------------------------------------------------

def rules64(logits, kw, V):
    """(seen, count, allowed, per-row values in 64 bits) on the CPU, token by token."""
    R = logits.shape[0]
    seen = torch.zeros(R, V, dtype=torch.bool)
    count = torch.zeros(R, V, dtype=torch.float64)
    if kw.get("history") is not None:
        h = kw["history"].cpu()
        col = lambda k, d: kw[k].cpu().tolist() if kw.get(k) is not None else d  # noqa: E731
        which, begin = col("hist_row", list(range(R))), col("hist_begin", [0] * R)
        end = col("hist_end", [h.shape[1]] * R)
        gb = col("gen_begin", begin)
        for r in range(R):
            if not 0 <= which[r] < h.shape[0]:
                continue
            for k in range(max(0, begin[r]), min(h.shape[1], end[r])):
                t = int(h[which[r], k])
                if 0 <= t < V:
                    seen[r, t] = True
                    count[r, t] += k >= gb[r]
    ok = torch.ones(R, V, dtype=torch.bool)
    m = kw.get("mask")
    if m is not None:
        m = m.cpu()
        m = m[None] if m.dim() == 1 else m
        if m.dtype == torch.int32:
            m = ((m.long()[:, :, None] >> torch.arange(32)) & 1).reshape(m.shape[0], -1)[:, :V]
        m = m != 0
        for r in range(R):
            j = int(kw["mask_row"][r]) if kw.get("mask_row") is not None else (r if m.shape[0] > 1 else 0)
            if 0 <= j < m.shape[0]:
                ok[r] = m[j]
    per = lambda k, d: (kw[k].cpu().double()[:, None] if isinstance(kw.get(k), torch.Tensor) else torch.full((R, 1), float(kw.get(k, d))).double())  # noqa: E731
    # scalars reach the kernel as 32-bit numbers
    per32 = lambda k, d: per(k, d).float().double()  # noqa: E731
    return seen, count, ok, per32("repetition", 1.0), per32("presence", 0.0), per32("frequency", 0.0), per32("temperature", 1.0)


def check_shape(logits, out, kw):
    V = logits.shape[1]
    seen, count, ok, rep, pres, freq, temp = rules64(logits, kw, V)
    l = logits.cpu().double()
    x = torch.where(seen, torch.where(l > 0, l / rep, l * rep), l)
    pen = freq * count + pres * (count > 0)
    b = kw["bias"].cpu().double() if kw.get("bias") is not None else torch.zeros(1, dtype=torch.float64)
    want = torch.where(ok, (x - pen + b) / temp, -INF)
    got = out.cpu().double()
    size = (x.abs() + 2 * pen.abs() + b.abs()) / temp
    # x/rep, freq*c, + pres, -, + bias, 1/T, * : at most 7 roundings of something no larger than `size`
    tol = half(out.dtype) * (want.abs() + 8 * U * size) + 8 * U * size + floor_of(out.dtype)
    fine = torch.isfinite(want)
    # a value that rounds beyond the type's range is infinite on both sides
    big = want.abs() >= torch.finfo(out.dtype).max * (1 - half(out.dtype))
    assert torch.equal(got[~fine & ok].isnan(), want[~fine & ok].isnan())
    assert torch.all(got[~ok] == -INF)
    sel = fine & ~big
    assert torch.all((got[sel] - want[sel]).abs() <= tol[sel]), float(((got[sel] - want[sel]).abs() / tol[sel].clamp(min=1e-300)).max())


def make_rules(g, R, V, L, mask, bias, layout, per_row=True, tokens=torch.int64):
    kw = {}
    if L:
        H = R if layout != "rows_of_others" else max(1, R // 2)
        tok = torch.randint(-2, V + 3, (H, L), generator=g, device="cuda")     # ids below 0 and beyond the vocabulary are padding
        tok[:, ::3] = torch.randint(0, max(1, V // 8), (H, len(range(0, L, 3))), generator=g, device="cuda")
        tok = tok.to(tokens)
        if layout == "time":
            tok = tok.t().contiguous().t()
        if layout == "apart":
            wide = torch.zeros(H, 2 * L + 3, dtype=tokens, device="cuda")
            wide[:, 1:2 * L + 1:2] = tok
            tok = wide[:, 1:2 * L + 1:2]
        kw["history"] = tok
        i32 = lambda lo, hi: torch.randint(lo, hi, (R,), generator=g, device="cuda").int()  # noqa: E731
        if layout == "rows_of_others":
            kw["hist_row"] = i32(-1, H + 1)                                     # some rows have no history row
        kw["hist_begin"] = i32(-2, L // 2 + 1)
        kw["hist_end"] = i32(0, L + 3)                                          # some before begin: an empty history
        kw["gen_begin"] = kw["hist_begin"] + i32(-1, L // 2 + 2)
    f = lambda lo, hi: (lo + (hi - lo) * torch.rand(R, generator=g, device="cuda"))  # noqa: E731
    if per_row:
        kw.update(repetition=f(0.7, 1.6), presence=f(-0.5, 0.9), frequency=f(-0.2, 0.4), temperature=f(0.3, 2.0))
    else:
        kw.update(repetition=1.3, presence=0.25, frequency=0.125, temperature=0.8)
    if bias == "shared":
        kw["bias"] = randn(g, V)
    elif bias == "row":
        kw["bias"] = randn(g, R, V + 5)[:, :V]
    if mask != "none":
        n = R
        if mask.endswith("_picked"):
            n = max(1, R // 3)
            kw["mask_row"] = torch.randint(-1, n + 1, (R,), generator=g, device="cuda").int()
        ok = torch.rand(n, V, generator=g, device="cuda") < 0.5
        if n > 2:
            ok[2] = False                                                       # a row its mask leaves nothing of
        if mask == "shared":
            kw["mask"] = ok[0]
        else:
            kw["mask"] = bits_of(ok) if mask.startswith("bits") else ok
    return kw


SHAPES = [(1, 1, 0, "none", "none", "rows"), (1, 2, 1, "bits", "none", "rows"), (3, 7, 5, "bytes", "shared", "time"),
          (5, 8, 17, "bits", "row", "rows_of_others"), (9, 31, 40, "bytes_picked", "none", "apart"), (4, 33, 0, "bits", "shared", "rows"),
          (6, 151, 300, "bits_picked", "row", "time"), (2, 2047, 64, "shared", "none", "rows"), (3, 8192, 700, "bits", "shared", "rows"),
          (2, 8193, 1000, "bytes", "row", "time"), (2, 20011, 513, "bits", "none", "rows_of_others"), (67, 129, 33, "bytes", "shared", "apart"),
          # enough rows for the workgroups with longer parts: several chunks, several rows a workgroup, short and long histories
          (90, 20011, 40, "bits", "shared", "rows"), (261, 4095, 33, "bytes", "none", "time"), (300, 3001, 120, "bits_picked", "none", "apart"),
          (262, 5000, 160, "bits", "row", "rows_of_others"), (257, 8200, 0, "bytes_picked", "shared", "rows"), (40, 2048, 9, "bits", "none", "rows")]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "-".join(map(str, c)))
def test_shape_logits(case, dtype):
    import ppo_amd
    R, V, L, mask, bias, layout = case
    g = gen(R * 1000 + V)
    kw = make_rules(g, R, V, L, mask, bias, layout, per_row=R != 4, tokens=torch.int32 if V % 2 else torch.int64)
    logits = (randn(g, R, V) * 3).to(dtype)
    before = logits.clone()
    out = ppo_amd.shape_logits(logits, **kw)
    assert out.dtype == dtype and torch.equal(logits, before)
    check_shape(logits, out, kw)
    # in place, and out of rows that lie apart at odd addresses: the same bits
    wide = torch.zeros(R, V + 3, dtype=dtype, device="cuda")
    wide[:, 1:V + 1] = logits
    view = wide[:, 1:V + 1]
    got = ppo_amd.shape_logits(view, out=view, **kw)
    assert got is view and torch.equal(view.float(), out.float())
    assert torch.all(wide[:, 0] == 0) and torch.all(wide[:, V + 1:] == 0)      # nothing beside the rows was touched


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "-".join(map(str, c)))
def test_shape_logits_backward(case, dtype):
    import ppo_amd
    R, V, L, mask, bias, layout = case
    g = gen(R * 2000 + V)
    kw = make_rules(g, R, V, L, mask, "none", layout, per_row=R != 4)
    logits, grad = (randn(g, R, V) * 3).to(dtype), randn(g, R, V).to(dtype)
    logits[0, 0] = 0.0
    bk = {k: v for k, v in kw.items() if k not in ("bias", "presence", "frequency", "gen_begin")}
    got = ppo_amd.shape_logits_backward(grad, logits, **bk)
    seen, _, ok, rep, _, _, temp = rules64(logits, kw, V)
    d = grad.cpu().double()
    want = torch.where(ok, torch.where(seen, torch.where(logits.cpu().double() > 0, d / rep, d * rep), d) / temp, 0.0)
    tol = (half(dtype) + 4 * U) * want.abs() * (1 + half(dtype)) + floor_of(dtype)      # 1/T, *, rep: 3 roundings
    assert torch.all((got.cpu().double() - want).abs() <= tol)
    both = grad.clone()
    assert ppo_amd.shape_logits_backward(both, logits, out=both, **bk) is both and torch.equal(both.float(), got.float())


def test_shape_backward_is_the_difference_quotient():
    """The forward is piecewise linear in each logit: a difference away from 0 gives the slope itself."""
    import ppo_amd
    g = gen(5)
    R, V = 4, 300
    kw = make_rules(g, R, V, 50, "bits", "shared", "rows")
    # powers of two in the rules and logits on a grid: the forward is exact in 32 bits, and so is its slope
    kw.update(repetition=2.0, presence=0.5, frequency=0.25, temperature=0.5, bias=torch.round(kw["bias"] * 8) / 8)
    x = torch.round(randn(g, R, V) * 8) / 8
    x = torch.where(x == 0, 0.125, x)
    h = 2.0 ** -5
    y0, y1 = (ppo_amd.shape_logits(x + s * h, **kw) for s in (-1, 1))
    slope = torch.where(torch.isfinite(y0), (y1 - y0) / (2 * h), 0.0)
    bk = {k: v for k, v in kw.items() if k not in ("bias", "presence", "frequency", "gen_begin")}
    assert torch.equal(ppo_amd.shape_logits_backward(torch.ones_like(x), x, **bk), slope)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_shape_masked_places_may_hold_anything(dtype):
    import ppo_amd
    g = gen(11)
    R, V = 6, 1000
    ok = torch.rand(R, V, generator=g, device="cuda") < 0.4
    x = randn(g, R, V).to(dtype)
    junk = torch.tensor([math.nan, INF, -INF, torch.finfo(dtype).min, torch.finfo(dtype).max], device="cuda").to(dtype)
    x = torch.where(ok, x, junk[torch.randint(0, 5, (R, V), generator=g, device="cuda")])
    out = ppo_amd.shape_logits(x, mask=ok, temperature=0.5)
    assert torch.all(out[~ok] == -INF) and torch.equal(out[ok].float(), (x[ok].float() * 2).to(dtype).float())
    grad = torch.where(ok, randn(g, R, V), math.nan).to(dtype)
    d = ppo_amd.shape_logits_backward(grad, x, mask=bits_of(ok), temperature=0.5)
    assert torch.all(d[~ok] == 0) and torch.equal(d[ok].float(), (grad[ok].float() * 2).to(dtype).float())
    # unmasked non-finite values go through
    y = torch.tensor([[math.nan, INF, -INF, 1.0]], device="cuda").to(dtype)
    z = ppo_amd.shape_logits(y, history=torch.tensor([[1, 2, 3]], device="cuda"), repetition=2.0)
    assert z[0, 0].isnan() and z[0, 1] == INF and z[0, 2] == -INF and z[0, 3] == 0.5


def test_shape_counts_a_token_seen_very_often():
    import ppo_amd
    L = 200001
    hist = torch.zeros(2, L, dtype=torch.int32, device="cuda")
    hist[1, ::2] = 5
    x = torch.zeros(2, 9, device="cuda")
    out = ppo_amd.shape_logits(x, history=hist, frequency=1.0, presence=0.5)
    assert out[0, 0] == -(L + 0.5) and out[1, 0] == -(L // 2 + 0.5) and out[1, 5] == -(L // 2 + 1 + 0.5) and out[1, 1] == 0


def test_history_of_a_buffer_is_its_actions_column():
    """Token histories read in place from the buffer's time-major actions."""
    import numpy as np
    import ppo_amd
    N, T, V = 5, 12, 40
    rng = np.random.RandomState(3)
    buf = ppo_amd.ExperienceBuffer(N, 2, T)
    acts = rng.randint(0, V, (T, N)).astype(np.uint64)
    z = np.zeros((T, N), np.float32)
    buf.add_many(np.zeros((T, N, 2), np.float32), z, acts, z, z.astype(np.uint8), z)
    hist = buf.stream_view("actions").view(T, N).t()
    g = gen(1)
    x = randn(g, N, V)
    begin = torch.tensor([0, 3, 12, 5, 1], device="cuda", dtype=torch.int32)
    kw = dict(history=hist, hist_begin=begin, repetition=1.5, frequency=0.3, presence=0.1)
    check_shape(x, ppo_amd.shape_logits(x, **kw), kw)
    buf.close()


# ---- statistics and objective ---------------------------------------------------------------------------------------------

def softmax64(logits, actions):
    """Per row in 64 bits: m, ln s, t/s, neglogp, entropy, p, ln p, and the roundings that s and t carry."""
    x = logits.double()
    V = x.shape[1]
    m = x.amax(1, keepdim=True)
    d = torch.where(x == -INF, -INF, x - m)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    dz = torch.where(e > 0, d, 0.0)
    p = e / s
    ts = (p * dz).sum(1)
    lns = s.log()[:, 0]
    a = actions.clamp(0, V - 1)[:, None]
    d_a = d.gather(1, a)[:, 0]
    nlp, ent = lns - d_a, lns - ts
    # a term e^d is off by 3 |d| u (difference, product, constant) + 2 u (exponential); terms are added one after the other
    # in a lane (V / 64 at most, of 32-bit sums that only grow) and then in a tree, with a rebasing each
    adds = (V / 64 + 48) * U
    rel_s = 3 * U * (-ts) + 2 * U + adds
    err_ts = 3 * U * (p * dz * dz).sum(1) + (2 * U + adds + rel_s) * (-ts) + 2 * U * (-ts)
    # log2 s, the action's power of two, their difference and the factor ln 2: 2 u each way of what they are (an action that is
    # forbidden has neither)
    err_nlp = rel_s + 2 * U * (lns.abs() + torch.where(torch.isfinite(d_a), d_a.abs() + nlp.abs(), 0.0))
    err_ent = rel_s + err_ts + 2 * U * (lns.abs() + ts.abs() + ent.abs())
    return dict(m=m, d=d, p=p, lns=lns, ts=ts, nlp=nlp, ent=ent, rel_s=rel_s, err_ts=err_ts, err_nlp=err_nlp, err_ent=err_ent)


POLICY = [(1, 1), (1, 2), (3, 3), (300, 6), (257, 18), (130, 63), (131, 64), (129, 65), (70, 151), (33, 512), (17, 513), (9, 1000),
          (5, 2048), (6, 2049), (5, 4099), (4, 8192), (3, 8193), (3, 16385), (2, 32768), (2, 50001), (3, 65537), (2, 131072), (2, 131075),
          (1, 200003), (1000, 33), (130, 40), (129, 41), (77, 48), (99, 49), (66, 56), (65, 57), (450, 25), (67, 97), (91, 100), (45, 129), (130, 150),
          (29, 193), (23, 385), (50, 386), (21, 600), (19, 768), (18, 767), (17, 769)]


def policy_inputs(R, V, dtype, seed, padded=False):
    g = gen(seed)
    logits = (randn(g, R, V) * 2.5).to(dtype)
    a = torch.randint(0, V, (R,), generator=g, device="cuda")
    if padded:
        a[::3] = -1
    return g, logits, a


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V", POLICY)
def test_action_stats(R, V, dtype):
    import ppo_amd
    g, logits, a = policy_inputs(R, V, dtype, R + V, padded=R > 4)
    if V > 3:
        logits[R // 2, 1::2] = -INF                                            # forbidden tokens
        logits[R // 2, 0] = 1.0
        if a[R // 2] >= 0:
            a[R // 2] = 0
    nlp, ent = ppo_amd.action_stats(logits, a)
    w = softmax64(logits, a)
    real = a >= 0
    assert torch.all(nlp[~real] == 0) and torch.all(ent[~real] == 0)
    assert torch.all(((nlp.double() - w["nlp"]).abs() <= w["err_nlp"])[real])
    assert torch.all(((ent.double() - w["ent"]).abs() <= w["err_ent"])[real])
    # rows that lie apart at odd addresses
    wide = torch.full((R, V + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:V + 1] = logits
    n2, e2 = ppo_amd.action_stats(wide[:, 1:V + 1], a)
    assert torch.all(((n2.double() - w["nlp"]).abs() <= w["err_nlp"])[real]) and torch.all(((e2.double() - w["ent"]).abs() <= w["err_ent"])[real])


@pytest.mark.parametrize("V", [5, 64, 100, 700, 3000, 20000, 140000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_without_a_distribution(V, dtype):
    import ppo_amd
    g = gen(V)
    x = (randn(g, 9, V) * 2).to(dtype)
    x[0] = -INF                                                                 # everything forbidden
    x[1, V // 2] = math.nan
    x[2, V - 1] = INF
    x[3] = torch.finfo(dtype).min                                               # a mask of the type's lowest value: uniform
    x[4, 1:] = torch.finfo(dtype).min
    x[5, :] = math.nan
    a = torch.tensor([0, 0, 0, 1, 0, 0, V, -2, -1], device="cuda")              # 6, 7: outside the vocabulary, 8: padding
    nlp, ent = (t.cpu() for t in ppo_amd.action_stats(x, a))
    assert nlp[0] == INF and ent[0] == 0
    for r in (1, 2, 5, 6, 7):
        assert nlp[r].isnan() and ent[r].isnan(), r
    assert abs(nlp[3] - math.log(V)) <= 1e-5 and abs(ent[3] - math.log(V)) <= 1e-5
    assert nlp[4] == 0 and ent[4] == 0 and nlp[8] == 0 and ent[8] == 0
    x[5], x[6:] = 0.5, 0.25
    a[6:8] = 0
    keep = torch.tensor([0, 3, 4, 5, 6, 7, 8], device="cuda")
    b = batch_of(g, x[keep], a[keep])
    r = ppo_amd.policy_loss(x[keep].contiguous(), b.new_values, b)
    assert torch.all(r.dlogits[0] == 0) and torch.all(r.dlogits[6] == 0) and torch.all(torch.isfinite(r.dlogits.float()))
    assert torch.all(torch.isfinite(r.stats[[1, 2, 3, 5]])) and r.dvalues[6] == 0
    # NaN rows poison the statistics and their own gradient only
    b = batch_of(g, x, a)
    r = ppo_amd.policy_loss(x, b.new_values, b)
    for row in (1, 2):
        assert torch.all(r.dlogits[row].isnan())
    assert torch.all(torch.isfinite(r.dlogits[[0, 3, 4, 5, 6, 7, 8]].float())) and r.stats[0].isnan()


class Batch:
    pass


def batch_of(g, logits, a, clip=0.2):
    R = logits.shape[0]
    b = Batch()
    w = softmax64(logits, a)
    step = 0.3 * randn(g, R)
    near = ((step.exp() - 1).abs() - clip).abs() < 0.01                          # the clip border itself belongs to neither side
    step = torch.where(near, 0.8 * step, step)
    b.actions = a
    b.neglogps = torch.where(torch.isfinite(w["nlp"]), w["nlp"].float() + step, step)
    b.advantages, b.values = randn(g, R), randn(g, R)
    b.returns = b.values + 0.5 * randn(g, R)
    b.new_values = b.values + 0.2 * randn(g, R)
    return b


def loss64(logits, b, a, clip, ent_c, vf_c, n):
    """(stats, dlogits, dvalues, tolerances) in 64 bits; `a` >= 0 rows only count."""
    w = softmax64(logits, a)
    real = a >= 0
    A, old = b.advantages.double(), b.neglogps.double()
    ratio = torch.exp(old - w["nlp"])
    pg = torch.maximum(-A * ratio, -A * ratio.clamp(1 - clip, 1 + clip))
    free = ~((A > 0) & (ratio > 1 + clip) | (A < 0) & (ratio < 1 - clip))
    gain = torch.where(free, A * ratio, 0.0)
    v, v0, ret = b.new_values.double(), b.values.double(), b.returns.double()
    far = v0 + (v - v0).clamp(-clip, clip) - ret
    q1, q2 = (v - ret) ** 2, far ** 2
    dv = torch.where(q2 > q1, torch.where((v - v0).abs() > clip, 0.0, far), v - ret)
    lnp = torch.where(w["p"] > 0, w["p"].clamp(min=1e-320).log(), 0.0)
    hit = torch.zeros_like(w["p"]).scatter_(1, a.clamp(0, logits.shape[1] - 1)[:, None], 1.0)
    shape = lnp + w["ent"][:, None]
    d = (gain[:, None] * (w["p"] - hit) + ent_c * w["p"] * shape) / n
    d = torch.where(real[:, None], d, 0.0)
    rel_g = w["err_nlp"] + U * (old.abs() + w["nlp"].abs()) + 8 * U
    dist = torch.where(w["d"] == -INF, 0.0, w["d"].abs())
    size = w["p"] * (gain.abs()[:, None] + ent_c * (lnp.abs() + w["ent"].abs()[:, None] + dist + w["ts"].abs()[:, None])) / n
    tol = size * ((3 * dist + 24) * U + 2 * w["rel_s"][:, None]) + w["p"] * ent_c * w["err_ts"][:, None] / n \
        + (rel_g * gain.abs() / n)[:, None] * (w["p"] + hit)
    # where ln p + H cancels: x = l log2(e) - m2 is relative to a rounded m2 = m log2(e), off by at most u |m2|; that shift is taken
    # out of the constant term again, which rounds three times numbers of its size
    tol = tol + 4 * U * U * torch.where(torch.isfinite(w["m"]), w["m"].abs().clamp(max=4096.0), 0.0) * w["p"] * ent_c / n
    # a power of two below 2^-126 is returned as 0 by the hardware's exponential: off by less than 2^-126 times its factor
    tol = tol + 2.0 ** -126 * (gain.abs()[:, None] + ent_c * (lnp.abs() + w["ent"].abs()[:, None] + dist)) / n
    tol = tol + half(logits.dtype) * (d.abs() + tol) + floor_of(logits.dtype)
    keep = lambda t: torch.where(real, t, 0.0)  # noqa: E731
    terms = [keep(pg), keep(torch.maximum(q1, q2) / 2), keep(w["ent"]), keep((w["nlp"] - old) ** 2 / 2), keep(((ratio - 1).abs() > clip).double())]
    means = [t.sum() / n for t in terms]
    errs = [(keep(rel_g * pg.abs())).sum() / n + 4 * U * means[0].abs(), (terms[1] * 16 * U + keep(8 * U * (v.abs() + v0.abs() + ret.abs()) * (q1 + q2).sqrt())).sum() / n,
            keep(w["err_ent"]).sum() / n + 2 * U * means[2].abs(), keep((w["nlp"] - old).abs() * (w["err_nlp"] + U * (old.abs() + w["nlp"].abs()))).sum() / n + 4 * U * means[3],
            4 * U * means[4]]
    loss = means[0] + vf_c * means[1] - ent_c * means[2]
    stats = torch.stack([loss] + means)
    stol = torch.stack([errs[0] + vf_c * errs[1] + ent_c * errs[2] + 4 * U * loss.abs()] + errs)
    vtol = 8 * U * (v.abs() + v0.abs() + ret.abs()) * vf_c / n
    return stats, stol, d, tol, keep(dv) * vf_c / n, vtol, w


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V", POLICY)
def test_policy_loss(R, V, dtype):
    import ppo_amd
    padded = R > 4 and V % 2 == 1
    g, logits, a = policy_inputs(R, V, dtype, 3 * R + V, padded=padded)
    if V > 3:
        logits[R // 2, 1::2] = -INF
        logits[R // 2, 0] = 1.0
        if a[R // 2] >= 0:
            a[R // 2] = 0
    b = batch_of(g, logits, a)
    n = float((a >= 0).sum())
    n32 = 1.0 / float(torch.tensor(1.0 / n, dtype=F32))                          # the kernel scales gradients by the 32-bit 1 / n
    r = ppo_amd.policy_loss(logits, b.new_values, b, denom=n)
    stats, stol, d, tol, dv, vtol, w = loss64(logits, b, a, float(torch.tensor(0.2)), float(torch.tensor(0.01)), 0.5, n)
    assert abs(n32 / n - 1) <= U
    real = a >= 0
    assert torch.all(((r.neglogps.double() - w["nlp"]).abs() <= w["err_nlp"])[real]) and torch.all(r.neglogps[~real] == 0)
    assert torch.all(((r.entropies.double() - w["ent"]).abs() <= w["err_ent"])[real])
    assert torch.all((r.dlogits.double() - d).abs() <= tol), float(((r.dlogits.double() - d).abs() / tol.clamp(min=1e-300)).max())
    assert torch.all((r.dvalues.double() - dv).abs() <= vtol)
    assert torch.all((r.stats.double() - stats).abs() <= stol + U * stats.abs()), (r.stats, stats, stol)
    # twice the same, bit for bit; and with the gradient written over the logits
    again = logits.clone()
    r2 = ppo_amd.policy_loss(again, b.new_values, b, denom=n, out=again)
    assert r2.dlogits is again and torch.equal(again.float(), r.dlogits.float()) and torch.equal(r2.stats, r.stats)
    # rows that lie apart at odd addresses, nothing written beside them
    wide = torch.zeros(R, V + 3, dtype=dtype, device="cuda")
    dw = torch.full((R, V + 5), 7.0, dtype=dtype, device="cuda")
    wide[:, 1:V + 1] = logits
    r3 = ppo_amd.policy_loss(wide[:, 1:V + 1], b.new_values, b, denom=n, out=dw[:, 1:V + 1])
    assert torch.all((r3.dlogits.double() - d).abs() <= tol)
    assert torch.all(dw[:, 0] == 7) and torch.all(dw[:, V + 1:] == 7)


def test_policy_loss_gradient_against_differences():
    """Central differences of the 64-bit objective, along random directions."""
    import ppo_amd
    g, logits, a = policy_inputs(12, 37, F32, 8)
    b = batch_of(g, logits, a)
    r = ppo_amd.policy_loss(logits, b.new_values, b, clip=0.3, ent_coef=0.05, vf_coef=0.7)
    clip, ent_c, vf_c = (float(torch.tensor(c)) for c in (0.3, 0.05, 0.7))

    def f(x, v):
        c = Batch()
        c.__dict__.update(b.__dict__)
        c.new_values = v
        return loss64(x, c, a, clip, ent_c, vf_c, 12.0)[0][0]
    x, v, h = logits.double(), b.new_values.double(), 2.0 ** -14
    for k in range(4):
        dx, dvv = randn(g, 12, 37).double(), randn(g, 12).double()
        num = (f(x + h * dx, v) - f(x - h * dx, v)) / (2 * h)
        assert abs(num - (r.dlogits.double() * dx).sum()) <= 1e-5               # second-order term h^2, gradient sums of 444 32-bit values
        num = (f(x, v + h * dvv) - f(x, v - h * dvv)) / (2 * h)
        assert abs(num - (r.dvalues.double() * dvv).sum()) <= 1e-5


def test_policy_loss_empty():
    import ppo_amd
    b = Batch()
    e = torch.zeros(0, device="cuda")
    b.actions, b.values, b.neglogps, b.returns, b.advantages = e.long(), e, e, e, e
    r = ppo_amd.policy_loss(torch.zeros(0, 5, device="cuda"), e, b)
    assert r.dlogits.shape == (0, 5) and torch.all(r.stats == 0)
    n, h = ppo_amd.action_stats(torch.zeros(0, 5, device="cuda"), e.long())
    assert n.shape == (0,) and h.shape == (0,)
    assert ppo_amd.shape_logits(torch.zeros(0, 5, device="cuda")).shape == (0, 5)
    assert ppo_amd.shape_logits(torch.zeros(5, 0, device="cuda")).shape == (5, 0)


def test_captured_and_replayed():
    """Two graphs and eager calls between their replays; every replay against the eager result on its inputs."""
    import ppo_amd
    R, V = 6, 70001
    sets = []
    for seed in (1, 2):
        g, x, a = policy_inputs(R, V, BF16, seed)
        b = batch_of(g, x, a)
        kw = make_rules(g, R, V, 64, "bits", "shared", "rows")
        sets.append((x, a, b, kw))

    def work(x, a, b, kw):
        y = ppo_amd.shape_logits(x, **kw)
        n, h = ppo_amd.action_stats(x, a)
        r = ppo_amd.policy_loss(x, b.new_values, b)
        return [y, n, h, r.stats, r.dlogits, r.dvalues]
    want = [work(*s) for s in sets]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            work(*s)
    torch.cuda.current_stream().wait_stream(side)
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(work(*s))
        graphs.append(gr)
    for _ in range(3):
        for k in (0, 1):
            for t in outs[k]:
                t.zero_()
            graphs[k].replay()
        mid = work(*sets[0])
        torch.cuda.synchronize()
        for k in (0, 1):
            for t, u in zip(outs[k], want[k]):
                assert torch.equal(t.float(), u.float())
        for t, u in zip(mid, want[0]):
            assert torch.equal(t.float(), u.float())


def test_on_another_stream():
    import ppo_amd
    g, x, a = policy_inputs(50, 4000, F32, 3)
    b = batch_of(g, x, a)
    want = ppo_amd.policy_loss(x, b.new_values, b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s in (s1, s2):
        with torch.cuda.stream(s):
            y = x * 1.0
            got.append(ppo_amd.policy_loss(y, b.new_values, b))
    torch.cuda.synchronize()
    for r in got:
        assert torch.equal(r.dlogits, want.dlogits) and torch.equal(r.stats, want.stats)
    assert torch.cuda.current_device() == 0


def test_refusals_on_the_gpu():
    import ppo_amd
    from ppo_amd import PpoXpPanic
    x = torch.zeros(4, 10, device="cuda")
    a = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: ppo_amd.shape_logits(x.t()), lambda: ppo_amd.shape_logits(x.double()), lambda: ppo_amd.shape_logits(x, out=x.half()),
                 lambda: ppo_amd.shape_logits(x, repetition=0.0), lambda: ppo_amd.shape_logits(x, temperature=torch.ones(3, device="cuda")),
                 lambda: ppo_amd.shape_logits(x, hist_end=a.int()), lambda: ppo_amd.shape_logits(x, mask_row=a.int()),
                 lambda: ppo_amd.shape_logits(x, history=a), lambda: ppo_amd.shape_logits(x, history=a[None].expand(3, 4)),
                 lambda: ppo_amd.shape_logits(x, history=a[None].expand(4, 4), hist_end=a),
                 lambda: ppo_amd.shape_logits(x, bias=x.double()), lambda: ppo_amd.shape_logits(x, bias=x[:, :9]),
                 lambda: ppo_amd.shape_logits(x, mask=x > 0, mask_row=a), lambda: ppo_amd.shape_logits(x, mask=(x > 0)[:3]),
                 lambda: ppo_amd.shape_logits(x, mask=a.int()[:, None].expand(4, 2)), lambda: ppo_amd.shape_logits(x, mask=x),
                 lambda: ppo_amd.shape_logits_backward(x.half(), x), lambda: ppo_amd.shape_logits_backward(x[:2], x),
                 lambda: ppo_amd.shape_logits(x.expand(4, 10)[:1].expand(4, 10)),
                 lambda: ppo_amd.action_stats(x, a.int()), lambda: ppo_amd.action_stats(x, a[:3]), lambda: ppo_amd.action_stats(x, a.cpu())):
        with pytest.raises(PpoXpPanic):
            call()
    b = Batch()
    v = torch.zeros(4, device="cuda")
    b.actions, b.values, b.neglogps, b.returns, b.advantages = a, v, v, v, v
    for kw in (dict(clip=-1.0), dict(denom=0.0), dict(ent_coef=math.nan), dict(out=x.half()), dict(out=x[:2])):
        with pytest.raises(PpoXpPanic):
            ppo_amd.policy_loss(x, v, b, **kw)
    b.returns = v[:3]
    with pytest.raises(PpoXpPanic):
        ppo_amd.policy_loss(x, v, b)


# ---- what a caller's tensors are left as ----------------------------------------------------------------------------------

def test_written_in_place_is_seen_by_autograd():
    import ppo_amd
    g = gen(21)
    R, V = 4, 40
    x = randn(g, R, V).requires_grad_()
    z = torch.zeros(R, device="cuda")
    batch = batch_of(g, x.detach(), torch.zeros(R, dtype=torch.int64, device="cuda"))
    for write in (lambda y: ppo_amd.shape_logits(y, temperature=0.5, out=y),
                  lambda y: ppo_amd.shape_logits_backward(torch.ones_like(y), x.detach(), temperature=0.5, out=y),
                  lambda y: ppo_amd.policy_loss(y, z, batch, out=y)):
        y = x.exp()                                        # saves its output for the backward pass
        write(y)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        y = x.exp()                                        # ... and one that is only read stays good
        ppo_amd.shape_logits(y, temperature=0.5)
        ppo_amd.policy_loss(y, z, batch)
        y.sum().backward()
    with torch.inference_mode():
        y = x.exp()
        want = ppo_amd.shape_logits(y, temperature=0.5)
        assert torch.equal(ppo_amd.shape_logits(y, temperature=0.5, out=y), want)


def test_no_tokens_and_no_rows():
    import ppo_amd
    for R, V in ((0, 5), (3, 0), (0, 0)):
        x = torch.zeros(R, V, device="cuda")
        nlp, ent = ppo_amd.action_stats(x, torch.zeros(R, dtype=torch.int64, device="cuda"))
        assert nlp.shape == ent.shape == (R,) and torch.all(nlp == 0) and torch.all(ent == 0)
        assert ppo_amd.shape_logits(x).shape == (R, V)


def test_results_are_ordinary_tensors():
    """They share memory with a workspace but not with each other: copies, views, pickles and in-place changes are theirs alone."""
    import copy
    import ppo_amd
    g, x, a = policy_inputs(64, 50, F32, 5)
    z = torch.zeros(64, device="cuda")
    r = ppo_amd.policy_loss(x, z, batch_of(g, x, a))
    nlp, ent = ppo_amd.action_stats(x, a)
    parts = [r.stats, r.dvalues, r.neglogps, r.entropies, nlp, ent]
    before = [p.clone() for p in parts]
    for k, p in enumerate(parts):
        assert p.is_contiguous() and not p.requires_grad and p._base is None
        assert torch.equal(copy.deepcopy(p), before[k]) and torch.equal(p.reshape(-1, 1)[:, 0], before[k])
        p.add_(1.0)
        assert all(torch.equal(q, before[j]) for j, q in enumerate(parts) if j > k)
        assert torch.equal(p, before[k] + 1.0)
