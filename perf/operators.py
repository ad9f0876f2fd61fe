"""The token-policy operators around the experience buffer, as cases to be timed and compared.

One training iteration of a policy whose actions are tokens calls them in this order: `shape` (penalties for repeated tokens, bias,
mask and temperature on the logits of one acting step), `stats` (neglogp and entropy of the chosen actions, what add_experience
stores), `write` (observation rows to 8 or 4 bits as they enter the store), `read` (a shuffled minibatch of those rows), `loss` (the
clipped objective of the minibatch with its gradient) and `shape_grad` (that gradient on to the raw logits).

`run` with own = False computes them from elementary torch operations in 32 bits (quotients next to a rounding border in 64),
with own = True through ppo_amd's public calls.  `exact` evaluates the definitions in 64 bits.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
TOP = {"int8": 127.0, "int4": 7.0, "e4m3": 448.0}
CLIP, ENT, VF = 0.2, 0.01, 0.5     # the reference's ModelConfig defaults
KINDS = ("shape", "shape_grad", "stats", "loss", "write", "read")


def _case(kind, name=None, **kw):
    c = {"kind": kind, **kw}
    if name:
        c["name"] = name
    return c


def _shape(kind, rows, vocab, dtype, hist, mask, bias="none", per_row=True, layout="rows", name=None):
    return _case(kind, name, rows=rows, vocab=vocab, dtype=dtype, hist=hist, mask=mask, bias=bias, per_row=per_row, layout=layout)


def listed():
    return [
        # one acting step of 8 envs writing 1024-token sequences: the history is the buffer's time-major actions [T, N]
        _shape("shape", 8, 131072, "bf16", 1024, "bits", layout="time", name="shape_step_8"),
        # one step of a busy sampler: requests with penalties of their own, a shared bias, a grammar's bit mask
        _shape("shape", 256, 131072, "bf16", 2048, "bits", bias="shared", name="shape_step_256"),
        # legal-action masks of 4096 envs with an odd discrete action set: no history, one byte an action
        _shape("shape", 4096, 151, "f32", 0, "bytes", per_row=False, name="shape_actions"),
        # the learner's way back through the same rules, an odd vocabulary, rows of a shuffled minibatch
        _shape("shape_grad", 2048, 50001, "bf16", 2048, "bits", layout="minibatch", name="shape_grad_2048"),
        # neglogp and entropy of one acting step: few long rows
        _case("stats", "stats_step_8", rows=8, vocab=131072, dtype="f32", padded=False),
        # ... and of a whole rollout at once
        _case("stats", "stats_4096", rows=4096, vocab=32768, dtype="bf16", padded=False),
        # the minibatch of the buffer's benchmark (T=128, N=65536, 32 minibatches) with a discrete action set
        _case("loss", "loss_actions", rows=262144, vocab=18, dtype="f32", padded=False),
        # a token minibatch with padding rows and an odd vocabulary
        _case("loss", "loss_tokens", rows=4096, vocab=50001, dtype="bf16", padded=True),
        # one insert of 4096 envs' 64-wide observations
        _case("write", "write_step", rows=4096, width=64, dtype="f32", format="int8", group=64, back=False),
        # hidden states of a whole rollout, written and read back in order
        _case("write", "write_states", rows=32768, width=4096, dtype="bf16", format="e4m3", group=128, back=True),
        # one minibatch of 64-wide observations out of a store of two million
        _case("read", "read_minibatch", store=2097152, rows=262144, width=64, dtype="f32", format="int8", group=64),
        # hidden states in 4 bits, a ragged width
        _case("read", "read_states", store=65536, rows=16384, width=4100, dtype="bf16", format="int4", group=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(KINDS)
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if kind in ("shape", "shape_grad"):
        vocab = _log(rng, 16, 140000)
        rows = _log(rng, 1, max(2, min(8192, 33_000_000 // vocab)))
        hist = rng.choice((0, _log(rng, 1, 4096), _log(rng, 16, 4096)))
        hist = min(hist, 8_000_000 // rows)
        return _shape(kind, rows, vocab, dtype, hist, rng.choice(("none", "bits", "bytes")), rng.choice(("none", "shared", "row")),
                      rng.random() < 0.7, rng.choice(("rows", "time", "minibatch")))
    if kind in ("stats", "loss"):
        vocab = _log(rng, 2, 200000)
        cap = 200_000_000 // (2 if kind == "loss" else 1) // (BYTES[dtype] // 2)
        rows = _log(rng, 1, max(2, min(262144, cap // vocab)))
        return _case(kind, rows=rows, vocab=vocab, dtype=dtype, padded=rng.random() < 0.3)
    width = _log(rng, 8, 8192)
    rows = _log(rng, 1, max(2, min(262144, 60_000_000 // width)))
    fmt, group = rng.choice(("int8", "e4m3", "int4")), rng.choice((32, 64, 128, 256))
    if kind == "write":
        return _case(kind, rows=rows, width=width, dtype=dtype, format=fmt, group=group, back=fmt != "int8")
    return _case(kind, store=_log(rng, rows, 4 * rows + 1), rows=rows, width=width, dtype=dtype, format=fmt, group=group)


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logits(c, g):
    """Logits of a trained policy: a spread of a few units with some favoured tokens."""
    x = torch.randn(c["rows"], c["vocab"], generator=g, device="cuda")
    return x.mul_(2.5).to(TYPES[c["dtype"]])


def _ints(g, lo, hi, size, dtype=torch.int32):
    return torch.randint(lo, hi, size, generator=g, device="cuda", dtype=torch.int64).to(dtype)


def _prepare_shape(c, g):
    R, V, L = c["rows"], c["vocab"], c["hist"]
    s = {"kind": c["kind"], "logits": _logits(c, g)}
    if c["kind"] == "shape_grad":
        s["grad"] = (torch.randn(R, V, generator=g, device="cuda") * (1.0 / R)).to(TYPES[c["dtype"]])
    kw = {}
    if L:
        H = R if c["layout"] != "minibatch" else max(1, R // 3)
        # repeated tokens: small indices are much likelier than large ones
        tok = (torch.rand(H, L, generator=g, device="cuda").pow_(3.0) * V).long().clamp_(max=V - 1)
        if c["layout"] == "time":
            tok = tok.t().contiguous().t()                  # [T, N] actions, seen as one row per env
        kw["history"] = tok
        if c["layout"] == "minibatch":
            kw["hist_row"] = _ints(g, 0, H, (R,))
        end = _ints(g, 0, L + 1, (R,))
        kw["hist_end"] = end
        kw["hist_begin"] = (end * torch.rand(R, generator=g, device="cuda") * 0.3).int()
        kw["gen_begin"] = kw["hist_begin"] + ((end - kw["hist_begin"]) * torch.rand(R, generator=g, device="cuda")).int()
    if c["per_row"]:
        u = torch.rand(4, R, generator=g, device="cuda")
        if L:
            kw.update(repetition=(1.0 + 0.4 * u[0]).contiguous(), presence=(0.8 * u[1]).contiguous(), frequency=(0.3 * u[2]).contiguous())
        kw["temperature"] = (0.5 + u[3]).contiguous()
    else:
        if L:
            kw.update(repetition=1.2, presence=0.5, frequency=0.1)
        kw["temperature"] = 0.7
    if c["bias"] != "none":
        kw["bias"] = torch.randn(V if c["bias"] == "shared" else (R, V), generator=g, device="cuda") if c["bias"] == "shared" else \
            torch.randn(R, V, generator=g, device="cuda")
    if c["mask"] == "bits":
        m = _ints(g, -2**31, 2**31, (R, (V + 31) // 32))
    elif c["mask"] == "bytes":
        m = torch.rand(R, V, generator=g, device="cuda") < 0.6
    if c["mask"] != "none":
        if R > 5:
            m[5].zero_()                                    # a state that allows nothing
        kw["mask"] = m
    s["rules"] = kw
    return s


def _prepare_policy(c, g):
    R, V = c["rows"], c["vocab"]
    s = {"kind": c["kind"], "logits": _logits(c, g)}
    a = torch.randint(0, V, (R,), generator=g, device="cuda")
    if c["kind"] == "stats":
        if c["padded"] and R > 2:
            a[::7] = -1
        s["actions"] = a
        return s
    nlp = torch.cat([torch.logsumexp(x.float(), 1) for x in s["logits"].split(1024)]) - s["logits"].gather(1, a[:, None])[:, 0].float()
    step = 0.15 * torch.randn(R, generator=g, device="cuda")
    # a ratio within rounding of the clip border is either side's right: inputs keep a hundredth away from both
    near = ((step.exp() - 1).abs() - CLIP).abs() < 0.01
    step = torch.where(near, step * 0.8, step)
    s["old_neglogps"] = nlp + step
    real = R
    if c["padded"] and R > 2:
        a[::7] = -1
        real = R - (R + 6) // 7
    s["actions"], s["denom"] = a, float(real)
    s["advantages"] = torch.randn(R, generator=g, device="cuda")
    s["old_values"] = torch.randn(R, generator=g, device="cuda")
    s["values"] = s["old_values"] + 0.2 * torch.randn(R, generator=g, device="cuda")
    s["returns"] = s["old_values"] + 0.5 * torch.randn(R, generator=g, device="cuda")
    return s


def _rows(rows, width, g):
    """Hidden states: most channels near one, a few large."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    return x.mul_(torch.rand(width, generator=g, device="cuda").pow_(-0.3))


def _row_bytes(fmt, width):
    return (width + 1) // 2 if fmt == "int4" else width


def _empty_store(fmt, n, width, group):
    kind = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "int4": torch.uint8}[fmt]
    return (torch.zeros(n, _row_bytes(fmt, width), device="cuda", dtype=torch.uint8).view(kind),
            torch.zeros(n, (width + group - 1) // group, device="cuda"))


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] in ("shape", "shape_grad"):
        return _prepare_shape(c, g)
    if c["kind"] in ("stats", "loss"):
        return _prepare_policy(c, g)
    s = {"kind": c["kind"], "format": c["format"], "group": c["group"], "width": c["width"], "dtype": TYPES[c["dtype"]]}
    if c["kind"] == "write":
        s["rows"] = _rows(c["rows"], c["width"], g).to(TYPES[c["dtype"]])
        s["at"], s["back"] = c["rows"] // 2, c["back"]      # the next free rows of a ring that is partly full
        s["codes"], s["scales"] = _empty_store(c["format"], c["rows"] + s["at"], c["width"], c["group"])
        return s
    s["codes"], s["scales"] = _empty_store(c["format"], c["store"], c["width"], c["group"])
    for at in range(0, c["store"], 65536):
        n = min(65536, c["store"] - at)
        _plain_write(_rows(n, c["width"], g), s["codes"], s["scales"], at, c["format"], c["group"])
    s["index"] = torch.randperm(c["store"], generator=g, device="cuda")[:c["rows"]].int()
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------------

def _column(v, like):
    return v[:, None] if isinstance(v, torch.Tensor) else v


def _counted(kw, R, V):
    """(seen anywhere in the row's history, occurrences in its generated part), [R, V]."""
    tok = kw["history"]
    if "hist_row" in kw:
        tok = tok[kw["hist_row"].long()]
    pos = torch.arange(tok.shape[1], device="cuda")[None]
    inside = (pos >= kw["hist_begin"][:, None]) & (pos < kw["hist_end"][:, None])
    generated = inside & (pos >= kw["gen_begin"][:, None])
    at = torch.where(inside, tok, V)
    seen = torch.zeros(R, V + 1, device="cuda").scatter_(1, at, 1.0)[:, :V] > 0
    count = torch.zeros(R, V + 1, device="cuda").scatter_add_(1, at, generated.float())[:, :V]
    return seen, count


def _allowed(mask, V):
    if mask.dtype == torch.bool:
        return mask
    bits = (mask[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    return bits.reshape(mask.shape[0], -1)[:, :V] != 0


def _plain_shape(s):
    kw, l = s["rules"], s["logits"]
    R, V = l.shape
    x = l.float()
    if "history" in kw:
        seen, count = _counted(kw, R, V)
        rep = _column(kw["repetition"], x)
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - (_column(kw["frequency"], x) * count + _column(kw["presence"], x) * (count > 0))
    if "bias" in kw:
        x = x + kw["bias"]
    x = x / _column(kw["temperature"], x)
    if "mask" in kw:
        x = torch.where(_allowed(kw["mask"], V), x, -math.inf)
    return x.to(l.dtype)


def _plain_shape_grad(s):
    kw, l = s["rules"], s["logits"]
    R, V = l.shape
    d = s["grad"].float() / _column(kw["temperature"], l)
    if "history" in kw:
        seen, _ = _counted(kw, R, V)
        rep = _column(kw["repetition"], l)
        d = torch.where(seen, torch.where(l > 0, d / rep, d * rep), d)
    if "mask" in kw:
        d = torch.where(_allowed(kw["mask"], V), d, 0.0)
    return d.to(l.dtype)


def _softmax_parts(x, a):
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    logp = x - m - torch.log(z)
    p = e / z
    return p, logp, -logp.gather(1, a.clamp(min=0)[:, None])[:, 0], -(p * logp).sum(1)


def _plain_stats(s):
    a = s["actions"]
    _, _, nlp, ent = _softmax_parts(s["logits"].float(), a)
    real = a >= 0
    return {"neglogps": torch.where(real, nlp, 0.0), "entropies": torch.where(real, ent, 0.0)}


def _plain_loss(s):
    a, n = s["actions"], s["denom"]
    real = a >= 0
    p, logp, nlp, ent = _softmax_parts(s["logits"].float(), a)
    adv, old = s["advantages"], s["old_neglogps"]
    ratio = torch.exp(old - nlp)
    plain, clipped = -adv * ratio, -adv * ratio.clamp(1 - CLIP, 1 + CLIP)
    pg = torch.maximum(plain, clipped)
    g = torch.where(plain >= clipped, adv * ratio, 0.0)
    v, v0, ret = s["values"], s["old_values"], s["returns"]
    vc = v0 + (v - v0).clamp(-CLIP, CLIP)
    e1, e2 = v - ret, vc - ret
    vl = 0.5 * torch.maximum(e1 * e1, e2 * e2)
    dv = torch.where(e1 * e1 >= e2 * e2, e1, torch.where((v - v0).abs() <= CLIP, e2, 0.0))
    kl = 0.5 * (nlp - old).square()
    far = (ratio - 1).abs() > CLIP
    hit = torch.zeros_like(p).scatter_(1, a.clamp(min=0)[:, None], 1.0)
    d = (g[:, None] * (p - hit) + ENT * p * (logp + ent[:, None])) / n
    mean = lambda t: torch.where(real, t.double(), 0.0).sum() / n  # noqa: E731
    parts = [mean(pg), mean(vl), mean(ent), mean(kl), mean(far)]
    stats = torch.stack([parts[0] + VF * parts[1] - ENT * parts[2]] + parts).float()
    return {"stats": stats, "dlogits": torch.where(real[:, None], d, 0.0).to(s["logits"].dtype), "dvalues": torch.where(real, VF * dv / n, 0.0),
            "neglogps": torch.where(real, nlp, 0.0), "entropies": torch.where(real, ent, 0.0)}


def _plain_write(rows, codes, scales, at, fmt, group):
    n, width = rows.shape
    G = scales.shape[1]
    x = torch.nn.functional.pad(rows.float(), (0, G * group - width)).reshape(n, G, group)
    amax = x.abs().amax(2).double()
    if fmt == "e4m3":                                       # the smallest power of two that brings the group within the format's range
        mant, ex = torch.frexp(amax / TOP[fmt])
        s = torch.ldexp(torch.ones_like(amax), torch.where(mant == 0.5, ex - 1, ex))
    else:
        s = (amax / TOP[fmt]).float().double()
    s = torch.where(amax < 2.0 ** -110, 0.0, s)
    q = torch.where(s[:, :, None] > 0, x.double() / s[:, :, None], 0.0)     # 64 bits: quotients next to a rounding border
    scales[at:at + n] = s.float()
    if fmt == "e4m3":
        codes.view(torch.uint8)[at:at + n] = q.float().reshape(n, -1)[:, :width].to(torch.float8_e4m3fn).view(torch.uint8)
        return
    q = q.round().to(torch.int8).reshape(n, -1)[:, :width]
    if fmt == "int4":
        q = torch.nn.functional.pad(q, (0, width % 2)).reshape(n, -1, 2)
        q = ((q[:, :, 0] & 15) | (q[:, :, 1] << 4)).view(torch.uint8)
    codes[at:at + n] = q


def _values(codes, fmt, width):
    if fmt != "int4":
        return codes.float()
    b = codes.view(torch.int8)
    return torch.stack(((b << 4) >> 4, b >> 4), 2).reshape(codes.shape[0], -1)[:, :width].float()


def _plain_read(codes, scales, index, s):
    raw = codes.view(torch.uint8)[index].view(codes.dtype)
    wide = scales[index].repeat_interleave(s["group"], 1)[:, :s["width"]]
    return (_values(raw, s["format"], s["width"]) * wide).to(s["dtype"])


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def _run_own(s):
    import ppo_amd
    k = s["kind"]
    if k == "shape":
        return ppo_amd.shape_logits(s["logits"], **s["rules"])
    if k == "shape_grad":
        rules = {n: v for n, v in s["rules"].items() if n not in ("bias", "presence", "frequency", "gen_begin")}
        return ppo_amd.shape_logits_backward(s["grad"], s["logits"], **rules)
    if k == "stats":
        nlp, ent = ppo_amd.action_stats(s["logits"], s["actions"])
        return {"neglogps": nlp, "entropies": ent}
    if k == "loss":
        batch = ppo_amd.ExperienceBatch(observations=None, actions=s["actions"], values=s["old_values"], neglogps=s["old_neglogps"],
                                        returns=s["returns"], advantages=s["advantages"])
        r = ppo_amd.policy_loss(s["logits"], s["values"], batch, clip=CLIP, ent_coef=ENT, vf_coef=VF, denom=s["denom"])
        return {"stats": r.stats, "dlogits": r.dlogits, "dvalues": r.dvalues, "neglogps": r.neglogps, "entropies": r.entropies}
    store = ppo_amd.QuantizedRows.of(s["codes"], s["scales"], s["width"], s["format"], s["group"])
    if k == "read":
        return store.read(s["index"], dtype=s["dtype"])
    store.write(s["rows"], s["at"])
    if s["back"]:
        n = s["rows"].shape[0]
        return {"scales": s["scales"], "rows": store.read(slice(s["at"], s["at"] + n), dtype=s["dtype"])}
    return {"scales": s["scales"], "codes": s["codes"]}


def run(state):
    s = state
    if own:
        return _run_own(s)
    k = s["kind"]
    if k == "shape":
        return _plain_shape(s)
    if k == "shape_grad":
        return _plain_shape_grad(s)
    if k == "stats":
        return _plain_stats(s)
    if k == "loss":
        return _plain_loss(s)
    if k == "read":
        return _plain_read(s["codes"], s["scales"], s["index"].long(), s)
    _plain_write(s["rows"], s["codes"], s["scales"], s["at"], s["format"], s["group"])
    if s["back"]:
        at, n = s["at"], s["rows"].shape[0]
        return {"scales": s["scales"], "rows": _plain_read(s["codes"], s["scales"], torch.arange(at, at + n, device="cuda"), s)}
    return {"scales": s["scales"], "codes": s["codes"]}


def work(case):
    c = case
    es, k = BYTES[c["dtype"]], c["kind"]
    n = c["rows"]
    if k in ("write", "read"):
        store = n * (_row_bytes(c["format"], c["width"]) + 4 * ((c["width"] + c["group"] - 1) // c["group"]))
        values = n * c["width"] * es
        if k == "read":
            return {"bytes": store + values + 4 * n, "flops": 2 * n * c["width"]}
        return {"bytes": (store + values) * (2 if c["back"] else 1), "flops": 4 * n * c["width"]}
    V = c["vocab"]
    if k == "stats":
        return {"bytes": n * V * es + 16 * n, "flops": 6 * n * V}
    if k == "loss":
        return {"bytes": 2 * n * V * es + 44 * n, "flops": 14 * n * V}
    bytes_ = 2 * n * V * es + 4 * n * c["hist"]             # half of the history slots are inside, 8 bytes each
    bytes_ += {"none": 0, "bits": n * V // 8, "bytes": n * V}[c["mask"]]
    if k == "shape":
        bytes_ += {"none": 0, "shared": 4 * V, "row": 4 * n * V}[c["bias"]]
    return {"bytes": bytes_, "flops": 4 * n * V}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------

def _exact_rules(s, lo, hi):
    """For rows lo..hi: (repetition factor applies, generated occurrences, allowed), from a histogram over (row, token)."""
    kw, V = s["rules"], s["logits"].shape[1]
    n = hi - lo
    seen = torch.zeros(n, V, dtype=torch.bool, device="cuda")
    count = torch.zeros(n, V, dtype=torch.float64, device="cuda")
    if "history" in kw:
        L = kw["history"].shape[1]
        which = kw["hist_row"][lo:hi].long() if "hist_row" in kw else torch.arange(lo, hi, device="cuda")
        b, g, e = (kw[k][lo:hi].long() for k in ("hist_begin", "gen_begin", "hist_end"))
        cell = torch.arange(n, device="cuda").repeat_interleave(e - b)
        first = torch.cumsum(e - b, 0) - (e - b)
        place = torch.arange(cell.numel(), device="cuda") - first[cell] + b[cell]
        key = cell * V + kw["history"].reshape(-1, L)[which[cell], place]
        seen = torch.bincount(key, minlength=n * V).reshape(n, V) > 0
        count = torch.bincount(key[place >= g[cell]], minlength=n * V).reshape(n, V).double()
    ok = torch.ones(n, V, dtype=torch.bool, device="cuda")
    if "mask" in kw:
        m = kw["mask"][lo:hi]
        if m.dtype == torch.bool:
            ok = m
        else:
            v = torch.arange(V, device="cuda")
            ok = (m.long()[:, v // 32] >> (v % 32)) % 2 == 1
    per = lambda name: kw[name][lo:hi, None].double() if isinstance(kw[name], torch.Tensor) else float(kw[name])  # noqa: E731
    return seen, count, ok, per


def _exact_shape(s):
    kw, l = s["rules"], s["logits"]
    R, V = l.shape
    out = torch.empty(R, V, dtype=torch.float64, device="cuda")
    step = max(1, 40_000_000 // V)
    for lo in range(0, R, step):
        hi = min(R, lo + step)
        seen, count, ok, per = _exact_rules(s, lo, hi)
        x = l[lo:hi].double()
        if s["kind"] == "shape_grad":
            y = s["grad"][lo:hi].double()
            if "history" in kw:
                r = per("repetition")
                y = y * torch.where(seen, torch.where(x > 0, x * 0 + 1 / r, x * 0 + r), 1.0)
            y = torch.where(ok, y / per("temperature"), 0.0)
        else:
            y = x
            if "history" in kw:
                r = per("repetition")
                y = y * torch.where(seen, torch.where(x > 0, x * 0 + 1 / r, x * 0 + r), 1.0)
                y = y - per("frequency") * count - torch.where(count > 0, x * 0 + per("presence"), 0.0)
            if "bias" in kw:
                y = y + (kw["bias"] if kw["bias"].dim() == 1 else kw["bias"][lo:hi]).double()
            y = torch.where(ok, y / per("temperature"), -math.inf)
        out[lo:hi] = y
    return out


def _exact_policy(s):
    l, a = s["logits"], s["actions"]
    R, V = l.shape
    real, at = a >= 0, a.clamp(min=0)
    nlp, ent = (torch.empty(R, dtype=torch.float64, device="cuda") for _ in range(2))
    d = torch.empty(R, V, dtype=torch.float64, device="cuda") if s["kind"] == "loss" else None
    step = max(1, 40_000_000 // V)
    for lo in range(0, R, step):
        hi = min(R, lo + step)
        x = l[lo:hi].double()
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        nlp[lo:hi] = -logp[torch.arange(hi - lo, device="cuda"), at[lo:hi]]
        ent[lo:hi] = torch.special.entr(p).sum(1)
        if d is not None:
            ratio = torch.exp(s["old_neglogps"][lo:hi].double() - nlp[lo:hi])
            A = s["advantages"][lo:hi].double()
            held = torch.where(A >= 0, ratio > 1 + CLIP, ratio < 1 - CLIP)     # the clipped branch is the larger one
            gain = torch.where(held, 0.0, A * ratio)[:, None]
            y = gain * p + ENT * p * (logp + ent[lo:hi, None])
            y[torch.arange(hi - lo, device="cuda"), at[lo:hi]] -= gain[:, 0]
            d[lo:hi] = torch.where(real[lo:hi, None], y / s["denom"], 0.0)
    keep = lambda t: torch.where(real, t, 0.0)  # noqa: E731
    out = {"neglogps": keep(nlp), "entropies": keep(ent)}
    if d is None:
        return out
    n = s["denom"]
    A, old = s["advantages"].double(), s["old_neglogps"].double()
    ratio = torch.exp(old - nlp)
    pg = -torch.minimum(A * ratio, A * torch.clamp(ratio, 1 - CLIP, 1 + CLIP))
    v, v0, ret = (s[k].double() for k in ("values", "old_values", "returns"))
    far = v0 + torch.clamp(v - v0, -CLIP, CLIP) - ret
    use = far.abs() > (v - ret).abs()
    dv = torch.where(use, torch.where((v - v0).abs() > CLIP, 0.0, far), v - ret)
    parts = [keep(pg).sum() / n, keep(torch.where(use, far, v - ret).square() / 2).sum() / n, keep(ent).sum() / n,
             keep((nlp - old).square() / 2).sum() / n, keep(((ratio - 1).abs() > CLIP).double()).sum() / n]
    stats = torch.stack([parts[0] + VF * parts[1] - ENT * parts[2]] + parts)
    return {**out, "stats": stats, "dlogits": d, "dvalues": keep(dv) * VF / n}


def _exact_scales(x, fmt):
    amax = x.abs().amax(2)
    if fmt == "e4m3":
        s = torch.exp2(torch.ceil(torch.log2(amax / TOP[fmt]) - 1e-13))
    else:
        s = (amax / TOP[fmt]).float().double()              # the stored scale is a 32-bit number: its rounding is part of the format
    return torch.where(amax < 2.0 ** -110, 0.0, s)


def _exact_write(s):
    fmt, g, at = s["format"], s["group"], s["at"]
    n, width = s["rows"].shape
    G = s["scales"].shape[1]
    scales = torch.zeros(s["scales"].shape, dtype=torch.float64, device="cuda")
    values = torch.empty(n, width, dtype=torch.float64, device="cuda")
    step = max(1, 30_000_000 // width)
    for lo in range(0, n, step):
        hi = min(n, lo + step)
        x = torch.zeros(hi - lo, G * g, dtype=torch.float64, device="cuda")
        x[:, :width] = s["rows"][lo:hi].double()
        x = x.reshape(hi - lo, G, g)
        sc = _exact_scales(x, fmt)
        scales[at + lo:at + hi] = sc
        q = torch.where(sc[:, :, None] > 0, x / sc[:, :, None], 0.0)
        if fmt == "e4m3":                                   # three bits behind the point of each power of two, 2^-9 the least step
            unit = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
            q = torch.round(q / unit) * unit
        else:
            q = torch.round(q)
        values[lo:hi] = (q * sc[:, :, None] if s["back"] else q).reshape(hi - lo, -1)[:, :width]
    if s["back"]:
        return {"scales": scales, "rows": values}
    codes = torch.zeros(s["codes"].shape, dtype=torch.int8, device="cuda")
    codes[at:at + n] = values.to(torch.int8)
    return {"scales": scales, "codes": codes}


def _exact_read(s):
    j = s["index"].long()
    q = s["codes"].view(torch.uint8)[j]
    if s["format"] == "int4":
        q = torch.stack((q % 16, q // 16), 2).reshape(j.numel(), -1)[:, :s["width"]].double()
        q = torch.where(q > 7, q - 16, q)
    else:
        q = q.view(s["codes"].dtype).to(torch.float32).double()
    which = torch.arange(s["width"], device="cuda") // s["group"]
    return q * s["scales"][j][:, which].double()


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] in ("shape", "shape_grad"):
        return _exact_shape(s)
    if s["kind"] in ("stats", "loss"):
        return _exact_policy(s)
    return _exact_write(s) if s["kind"] == "write" else _exact_read(s)
