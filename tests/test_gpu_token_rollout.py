"""The token-policy operators together, as a training iteration uses them, and the buffer whose rows are quantised."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def streams(rng, T, N, D, V=11):
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return dict(obs=f(T, N, D), rewards=f(T, N), actions=rng.integers(0, V, (T, N)).astype(np.uint64), vals=f(T, N),
                dones=(rng.random((T, N)) < 0.1).astype(np.uint8), neglogps=np.abs(f(T, N)))


def step(r, t):
    return tuple(r[k][t] for k in ("obs", "rewards", "actions", "vals", "dones", "neglogps"))


@pytest.mark.parametrize("fmt,group,dtype", [("int8", 32, torch.float32), ("e4m3", 64, torch.bfloat16), ("int4", 16, torch.float16)])
@pytest.mark.parametrize("steps", [5, 8, 13, 21])       # below, at and past the capacity of 8, and past it twice over
def test_quantized_buffer_holds_the_ordinary_one(fmt, group, dtype, steps):
    import ppo_amd
    N, D, cap = 6, 37, 8
    r = streams(np.random.default_rng(steps), steps, N, D)
    plain = ppo_amd.ExperienceBuffer.new(N, D, cap)
    quant = ppo_amd.ExperienceBuffer.new_quantized(N, D, cap, fmt, group, dtype)
    many = ppo_amd.ExperienceBuffer.new_quantized(N, D, cap, fmt, group, dtype)
    cu = lambda a, t: torch.from_numpy(a.astype(np.int64 if t is torch.int64 else np.float32)).cuda()  # noqa: E731
    for t in range(steps):
        obs, rew, act, val, done, nlp = step(r, t)
        plain.add_experience(obs, rew, act, val, done, nlp)
        if t % 2:
            quant.add_experience(obs, rew, act, val, done, nlp)
        else:
            f = torch.float32
            quant.add_experience_device(cu(obs, f), cu(rew, f), cu(act, torch.int64), cu(val, f), cu(done, f), cu(nlp, f))
    many.add_many(r["obs"], r["rewards"], r["actions"], r["vals"], r["dones"], r["neglogps"])
    obs, act, val, nlp = plain.training_views()
    M = len(plain) * N
    store = ppo_amd.QuantizedRows(M, D, fmt, group)
    store.write(obs)
    want = store.read(dtype=dtype)
    for b in (quant, many):
        o, a, v, n = b.training_views()
        assert torch.equal(o, want) and torch.equal(a, act) and torch.equal(v, val) and torch.equal(n, nlp)
    last = np.zeros(N, np.uint8)
    ret = plain.returns(last)
    assert torch.equal(quant.returns(last), ret) and torch.equal(many.returns(last), ret)
    for B in (M, 7, max(1, M // 2)):
        for kw in (dict(seed=3), dict(seed=4, device_shuffle=True), dict(seed=5, bijection=True),
                   dict(perm=torch.randperm(M, generator=gen(1), device="cuda").int())):
            for streaming in (False, True):
                plain.set_streaming(streaming)
                quant.set_streaming(streaming)
                a = ppo_amd.ExperienceBatcher(plain, B).into_iter(**kw)
                b = ppo_amd.ExperienceBatcher(quant, B).into_iter(**kw)
                perm = torch.from_numpy(b.perm().astype(np.int64)).cuda()
                count = 0
                for k, (x, y) in enumerate(zip(a, b)):
                    at = min(k * B, M - B)
                    assert torch.equal(y.observations, want[perm[at:at + B]]) and y.observations.dtype == dtype
                    for name in ("actions", "values", "neglogps", "returns"):
                        assert torch.equal(getattr(x, name), getattr(y, name))
                    # the advantages of a different gather route may differ in the last bit of the mean and deviation
                    assert torch.allclose(x.advantages, y.advantages, rtol=1e-5, atol=1e-5)
                    count += 1
                assert count == -(-M // B)
    quant.set_streaming(False)
    it = ppo_amd.ExperienceBatcher(quant, 7).into_iter(seed=1)
    with pytest.raises(ppo_amd.PpoXpPanic):
        it.next_host()
    with pytest.raises(ppo_amd.PpoXpPanic):
        next(it.host_batches())
    for b in (plain, quant, many):
        b.close()


def test_quantized_buffer_refusals():
    import ppo_amd
    b = ppo_amd.ExperienceBuffer.new_quantized(4, 16, 3)
    z, zi = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for obs in (torch.zeros(4, 15, device="cuda"), torch.zeros(3, 16, device="cuda"), torch.zeros(4, 16), torch.zeros(4, 16, device="cuda").double()):
        with pytest.raises(ppo_amd.PpoXpPanic):
            b.add_experience_device(obs, z, zi, z, z, z)
    n = np.zeros(4, np.float32)
    with pytest.raises(ppo_amd.PpoXpPanic):
        b.add_experience(np.zeros((4, 15), np.float32), n, n.astype(np.uint64), n, n.astype(np.uint8), n)
    assert len(b) == 0
    with pytest.raises(ppo_amd.PpoXpPanic):
        ppo_amd.ExperienceBuffer.new_quantized(4, 16, 3, format="int2")
    b.close()


def shaped64(l, seen, count, ok, rep, pres, freq, temp):
    x = torch.where(seen, torch.where(l > 0, l / rep, l * rep), l) - (freq * count + pres * (count > 0))
    return torch.where(ok, x / temp, -math.inf)


def test_one_training_iteration():
    """Act under rules whose history is the buffer's own actions, store neglogps and quantised states, and learn from shuffled
    minibatches: the distribution the learner sees is the one that acted, and the gradient on the raw logits is the 64-bit one."""
    import ppo_amd
    T, N, V, D, B = 9, 7, 150, 64, 20
    g = gen(77)
    rules = dict(repetition=1.3, presence=0.2, frequency=0.1, temperature=0.7)
    W = torch.randn(D, V, generator=g, device="cuda") * 0.3
    ok = torch.rand(N, V, generator=g, device="cuda") < 0.7          # one mask per env
    ok[:, 0] = True
    buf = ppo_amd.ExperienceBuffer.new_quantized(N, D, T, "int8", 32)
    begin = torch.zeros(N, dtype=torch.int32, device="cuda")          # where the env's running episode starts
    begins = torch.zeros(T, N, dtype=torch.int32, device="cuda")
    done = torch.zeros(N, device="cuda")
    probe = ppo_amd.QuantizedRows(N, D, "int8", 32)
    for t in range(T):
        begin = torch.where(done > 0, t, begin).int()
        begins[t] = begin
        states = torch.randn(N, D, generator=g, device="cuda")
        probe.write(states)                                           # act on the states as the learner will read them
        logits = probe.read() @ W
        hist = buf.stream_view("actions").view(len(buf), N).t() if t else None
        kw = dict(history=hist, hist_begin=begin, hist_end=torch.full_like(begin, t)) if t else {}
        x = ppo_amd.shape_logits(logits, mask=ok, **rules, **kw)
        assert torch.all(x[~ok] == -math.inf)
        a = torch.multinomial(torch.softmax(x, 1), 1, generator=g)[:, 0]
        nlp, ent = ppo_amd.action_stats(x, a)
        assert torch.all(torch.isfinite(nlp)) and torch.all(ent > 0)
        buf.add_experience_device(states, torch.randn(N, generator=g, device="cuda"), a, torch.randn(N, generator=g, device="cuda"), done, nlp)
        done = (torch.rand(N, generator=g, device="cuda") < 0.2).float()
    buf.returns(done.cpu().numpy().astype(np.uint8))
    M = T * N
    it = ppo_amd.ExperienceBatcher(buf, B).into_iter(seed=5, bijection=True)
    perm = torch.from_numpy(it.perm().astype(np.int64)).cuda()
    hist = buf.stream_view("actions").view(T, N).t()
    for k, batch in enumerate(it):
        at = min(k * B, M - B)
        idx = perm[at:at + B]
        e, t = idx % N, idx // N
        kw = dict(history=hist, hist_row=e.int(), hist_begin=begins[t, e], hist_end=t.int(), mask=ok, mask_row=e.int(), temperature=0.7, repetition=1.3)
        logits = batch.observations @ W
        x = ppo_amd.shape_logits(logits, presence=0.2, frequency=0.1, **kw)
        values = batch.values + 0.1
        batch.neglogps = batch.neglogps.clone()
        nlp, _ = ppo_amd.action_stats(x, batch.actions)
        # the same rows, the same rules: products of 64 terms in another order of a batch of another size, 2^-24 each, on logits of
        # up to 20, divided by the temperature
        assert torch.all((nlp - batch.neglogps).abs() <= 64 * 20 / 0.7 * 2.0 ** -23)
        batch.neglogps += 0.15 * torch.where(torch.arange(B, device="cuda") % 2 == 0, 1.0, -1.0)
        r = ppo_amd.policy_loss(x, values, batch, ent_coef=0.03)
        d = ppo_amd.shape_logits_backward(r.dlogits, logits, **kw)
        # 64 bits, by autograd on the CPU
        l = logits.cpu().double().requires_grad_()
        seen, count = torch.zeros(B, V, dtype=torch.bool), torch.zeros(B, V, dtype=torch.float64)
        h, bg = hist.cpu(), begins.cpu()
        for j in range(B):
            for s in range(int(bg[t[j], e[j]]), int(t[j])):
                seen[j, h[e[j], s]] = True
                count[j, h[e[j], s]] += 1
        c32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
        y = shaped64(l, seen, count, ok.cpu()[e.cpu()], c32(1.3), c32(0.2), c32(0.1), c32(0.7))
        logp = torch.log_softmax(y, 1)
        nlp64 = -logp[torch.arange(B), batch.actions.cpu()]
        p = logp.exp()
        ent64 = -(p * torch.where(p > 0, logp, 0.0)).sum(1)
        A = batch.advantages.cpu().double()
        ratio = torch.exp(batch.neglogps.cpu().double() - nlp64)
        lo, hi = 1 - c32(0.2), 1 + c32(0.2)
        assert torch.all(((ratio - lo).abs() > 1e-3) & ((ratio - hi).abs() > 1e-3))
        loss = torch.maximum(-A * ratio, -A * ratio.clamp(lo, hi)).mean() - c32(0.03) * ent64.mean()
        loss.backward()
        want = l.grad
        # the shaped logits carry up to 8 roundings of numbers below 40, which move each probability by 8 * 40 * 2^-24 of itself
        rel = 8 * 40 * 2.0 ** -24 + 64 * 2.0 ** -24
        assert (d.cpu().double() - want).norm() <= 4 * rel * want.norm()
        assert torch.all(d[~ok[e]] == 0)
    buf.close()
