"""The documented loop of a token policy over a buffer of quantised rows: acting, learning, and the gradients it leaves in the model."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
num_envs, obs_size, capacity, vocab, batch_size = 5, 32, 7, 90, 12


class Env:
    def __init__(self, g):
        self.g = g

    def step(self, actions):
        r = lambda *s: torch.rand(*s, generator=self.g, device="cuda")  # noqa: E731
        return r(num_envs, obs_size) - 0.5, r(num_envs), (r(num_envs) < 0.2).float()


def test_documented_loop():
    import ppo_amd
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    w = (torch.randn(obs_size, vocab, generator=g, device="cuda") * 0.4).requires_grad_()
    c = (torch.randn(obs_size, generator=g, device="cuda") * 0.4).requires_grad_()
    model = lambda o: (o @ w, o @ c)  # noqa: E731
    env = Env(g)
    obs, rewards, dones = env.step(None)
    legal = torch.rand(num_envs, vocab, generator=g, device="cuda") < 0.8
    epoch = 1

    buf = ppo_amd.ExperienceBuffer.new_quantized(num_envs, obs_size, capacity, format="int8", group=64)
    rules = dict(repetition=1.1, temperature=0.7)
    first = torch.zeros(num_envs, dtype=torch.int32, device="cuda")
    firsts = torch.zeros(capacity, num_envs, dtype=torch.int32, device="cuda")
    for t in range(capacity):
        firsts[t] = first
        seen = dict(history=buf.stream_view("actions").view(t, num_envs).t(), hist_begin=first) if t else {}
        with torch.no_grad():
            logits, values = model(obs)
        x = ppo_amd.shape_logits(logits, mask=legal, **rules, **seen)
        actions = torch.multinomial(torch.softmax(x.float(), 1), 1, generator=g)[:, 0]
        assert torch.all(legal.gather(1, actions[:, None]))
        neglogps, entropies = ppo_amd.action_stats(x, actions)
        buf.add_experience_device(obs, rewards, actions, values, dones, neglogps)
        obs, rewards, dones = env.step(actions)
        first = torch.where(dones > 0, t + 1, first)
    buf.returns(dones.cpu().numpy().astype("uint8"))
    it = ppo_amd.ExperienceBatcher(buf, batch_size).into_iter(seed=epoch)
    perm = torch.from_numpy(it.perm().astype("int64")).cuda()
    history = buf.stream_view("actions").view(capacity, num_envs).t()
    count = 0
    for k, batch in enumerate(it):
        at = min(k * batch_size, perm.numel() - batch_size)
        step, row = perm[at:at + batch_size] // num_envs, perm[at:at + batch_size] % num_envs
        seen = dict(history=history, hist_row=row.int(), hist_begin=firsts[step, row], hist_end=step.int(), mask=legal, mask_row=row.int())
        logits, values = model(batch.observations)
        r = ppo_amd.policy_loss(ppo_amd.shape_logits(logits, **rules, **seen), values, batch, clip=0.2, ent_coef=0.01, vf_coef=0.5)
        dlogits = ppo_amd.shape_logits_backward(r.dlogits, logits, **rules, **seen)
        torch.autograd.backward([logits, values], [dlogits, r.dvalues])
        # the same in 64 bits by autograd
        o, W, C = batch.observations.cpu().double(), w.detach().cpu().double().requires_grad_(), c.detach().cpu().double().requires_grad_()
        l, v = o @ W, o @ C
        was = torch.zeros(batch_size, vocab, dtype=torch.bool)
        for j in range(batch_size):
            was[j, history[row[j], firsts[step[j], row[j]]:step[j]].cpu()] = True
        f32 = lambda y: float(torch.tensor(y, dtype=torch.float32))  # noqa: E731
        y = torch.where(was, torch.where(l > 0, l / f32(1.1), l * f32(1.1)), l) / f32(0.7)
        logp = torch.log_softmax(torch.where(legal[row].cpu(), y, -math.inf), 1)
        act = batch.actions.cpu()
        nlp = -logp[torch.arange(batch_size), act]
        ent = -(logp.exp() * torch.where(torch.isfinite(logp), logp, 0.0)).sum(1)
        A, old, ret, v0 = (q.cpu().double() for q in (batch.advantages, batch.neglogps, batch.returns, batch.values))
        ratio = torch.exp(old - nlp)
        assert torch.all((ratio - 1).abs() < 0.1)              # the rows as they read back are near those that acted
        far = v0 + (v - v0).clamp(-f32(0.2), f32(0.2)) - ret
        loss = (torch.maximum(-A * ratio, -A * ratio.clamp(0.8, 1.2)) + 0.25 * torch.maximum((v - ret) ** 2, far ** 2) - f32(0.01) * ent).mean()
        loss.backward()
        # logits below 16 from 32 products, shaped with 3 more roundings: off by 35 * 16 * 2^-24 each, which moves a probability by as much of
        # itself and the old neglogp's ratio too; the gradients of the model sum 12 rows of them
        rel = 4 * 35 * 16 * 2.0 ** -24
        assert (w.grad.cpu().double() - W.grad).norm() <= rel * W.grad.norm() and (c.grad.cpu().double() - C.grad).norm() <= rel * C.grad.norm()
        assert abs(r.stats[0].item() - loss.item()) <= rel * (loss.abs().item() + 1)
        w.grad, c.grad = None, None
        count += 1
    assert count == 3
    buf.close()
