"""No token of a row is lost: statistics and objective of rows whose probability lies on one token at each place where a kernel's
lanes, vectors, chunks or waves meet, and sums held to what the route's own additions can be off by.

A sum of non-negative terms is off by at most one u = 2^-24 of itself for each addition on a term's way: those of its lane one after
the other (LANE, by route) and then at most JOINS roundings in the trees of a wave and a workgroup, each preceded by a rebasing."""
import math

import pytest
import torch

from test_gpu_policy_ops import BF16, F16, F32, U, batch_of, gen, loss64, randn, softmax64

pytestmark = pytest.mark.gpu
JOINS = 48        # two trees of six additions, four rebasings (difference, power, product), the last of (s, t) in the log


def lane_terms(R, V, dtype, loss):
    """Additions in one lane, at most."""
    if V <= 2048:
        return 48                                           # elements of a lane in the turned and the group kernels
    if R < 128 and V > (65536 if loss else 98304):
        return 16 + V // 4096 // 64 + 1                     # two vectors a thread of a chunk, then chunks by 64 lanes
    if loss:
        beyond = V > (65536 if dtype == F32 else 131072) - 8
        return 3 * 8 * (V // 8192 + 1) if beyond else 128   # a vector of 8 and its rebasing every 8192 tokens; 16 vectors at most
    return 64 + 4 * (V // 8192 + 1)                         # eight vectors, and a join after each step


def tight(w, R, V, dtype, loss):
    """softmax64's errors of neglogp and entropy with the sum's share as above."""
    adds = (lane_terms(R, V, dtype, loss) + JOINS) * U
    ts, p, d = w["ts"], w["p"], torch.where(w["p"] > 0, w["d"], 0.0)
    rel_s = 3 * U * (-ts) + 2 * U + adds
    err_ts = 3 * U * (p * d * d).sum(1) + (2 * U + adds + rel_s) * (-ts) + 2 * U * (-ts)
    err_nlp = w["err_nlp"] - w["rel_s"] + rel_s
    err_ent = w["err_ent"] - w["rel_s"] - w["err_ts"] + rel_s + err_ts
    return err_nlp, err_ent


def seams(V):
    if V <= 2200:
        return list(range(V))
    at = {0, 1, V // 2, V - 1}
    for step in (512, 2048, 4096, 8192, 65536):             # a wave's vectors, 256 threads', a chunk, 1024 threads', a row's registers
        for m in list(range(0, V + 1, step))[-40:] + list(range(0, V + 1, step))[:20]:
            at |= {m - 9, m - 8, m - 1, m, m + 1, m + 7, m + 8}
    for k in range(1, 20):
        at |= {V - k, V - V % 8 - k, V - V % 8 + k % 8}
    return sorted(k for k in at if 0 <= k < V)


def held(got, want, err, name):
    over = (got.double() - want).abs() / err
    assert torch.all(over <= 1), (name, int(over.argmax()), float(over.max()))


SHORT = [(600, 5), (600, 18), (600, 47), (600, 48), (600, 49), (600, 63), (600, 64), (600, 65), (600, 100), (700, 151), (1100, 513), (2100, 2047), (2100, 2048),
         (335600, 50), (168100, 100), (112000, 150), (43700, 385), (22000, 765)]                   # ... and calls large enough to be turned
LONG = [(64, 2049), (64, 4095), (300, 4097), (64, 8191), (300, 8193), (64, 16385), (300, 20011), (64, 32768), (64, 32769), (300, 50001), (100, 65536),
        (100, 65537), (130, 70001), (100, 98305), (100, 131072), (100, 131075), (130, 140001), (60, 200003)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V", SHORT + LONG)
def test_no_token_is_lost(R, V, dtype):
    import ppo_amd
    places = seams(V)
    for k0 in range(0, max(len(places), 1), R):
        g = gen(V + k0)
        heavy = torch.tensor([places[(k0 + r) % len(places)] for r in range(R)], device="cuda")
        x = randn(g, R, V)
        x.scatter_(1, heavy[:, None], math.log(V) + 1.0)      # a third to a half of the row's probability
        x = x.to(dtype)
        a = torch.where(torch.arange(R, device="cuda") % 2 == 0, heavy, (heavy + 1) % V)
        w = softmax64(x, a)
        err_nlp, err_ent = tight(w, R, V, dtype, False)
        nlp, ent = ppo_amd.action_stats(x, a)
        held(nlp, w["nlp"], err_nlp, "neglogp")
        held(ent, w["ent"], err_ent, "entropy")
        b = batch_of(g, x, a)
        r = ppo_amd.policy_loss(x, b.new_values, b)
        err_nlp, err_ent = tight(w, R, V, dtype, True)
        held(r.neglogps, w["nlp"], err_nlp, "neglogp of the objective")
        held(r.entropies, w["ent"], err_ent, "entropy of the objective")
        stats, stol, d, tol, dv, vtol, _ = loss64(x, b, a, float(torch.tensor(0.2)), float(torch.tensor(0.01)), 0.5, float(R))
        assert torch.all((r.dlogits.double() - d).abs() <= tol)
        assert torch.all((r.dvalues.double() - dv).abs() <= vtol) and torch.all((r.stats.double() - stats).abs() <= stol + U * stats.abs())
        del d, tol, w, x, r


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V", [(64, 20011), (300, 50001), (100, 65537), (130, 70001), (100, 131075), (130, 140001), (60, 200003), (20, 600001)])
def test_sums_are_as_close_as_their_additions(R, V, dtype):
    """Rows whose probability is spread over all tokens: eight of them are more than the tolerance up to 200 000 tokens."""
    import ppo_amd
    g = gen(V)
    x = (randn(g, R, V) * 0.5).to(dtype)
    a = torch.randint(0, V, (R,), generator=g, device="cuda")
    w = softmax64(x, a)
    err_nlp, err_ent = tight(w, R, V, dtype, False)
    nlp, ent = ppo_amd.action_stats(x, a)
    held(nlp, w["nlp"], err_nlp, "neglogp")
    held(ent, w["ent"], err_ent, "entropy")
    b = batch_of(g, x, a)
    r = ppo_amd.policy_loss(x, b.new_values, b)
    err_nlp, err_ent = tight(w, R, V, dtype, True)
    held(r.neglogps, w["nlp"], err_nlp, "neglogp of the objective")
    held(r.entropies, w["ent"], err_ent, "entropy of the objective")


@pytest.mark.parametrize("V", [60, 151, 2049, 20011, 50001, 70001, 140001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_long_runs_of_forbidden_tokens(V, dtype):
    """Masks that leave runs of a row: whole lanes, waves and chunks hold nothing but -inf."""
    import ppo_amd
    for R in (40, 300):
        g = gen(V + R)
        x = (randn(g, R, V) * 2).to(dtype)
        first = torch.randint(0, V, (R,), generator=g, device="cuda")
        length = torch.randint(1, max(2, V // 3), (R,), generator=g, device="cuda")
        few = torch.arange(R, device="cuda") % 4 == 0
        length = torch.where(few, length.clamp(max=3), length)
        place = torch.arange(V, device="cuda")[None]
        ok = ((place - first[:, None]) % V) < length[:, None]
        x = torch.where(ok, x, -math.inf)
        a = torch.where(torch.arange(R, device="cuda") % 3 == 0, (first + length - 1) % V, first)
        w = softmax64(x, a)
        for loss in (False, True):
            err_nlp, err_ent = tight(w, R, V, dtype, loss)
            if loss:
                b = batch_of(g, x, a)
                r = ppo_amd.policy_loss(x, b.new_values, b)
                nlp, ent = r.neglogps, r.entropies
                _, _, d, tol, _, _, _ = loss64(x, b, a, float(torch.tensor(0.2)), float(torch.tensor(0.01)), 0.5, float(R))
                assert torch.all((r.dlogits.double() - d).abs() <= tol) and torch.all(r.dlogits[~ok] == 0)
            else:
                nlp, ent = ppo_amd.action_stats(x, a)
            held(nlp, w["nlp"], err_nlp, "neglogp")
            held(ent, w["ent"], err_ent, "entropy")
