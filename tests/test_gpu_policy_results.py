"""What the results of action_stats and policy_loss are as tensors: memory of their own, nothing of the call behind them."""
import io

import pytest
import torch

from test_gpu_policy_ops import BF16, F32, batch_of, policy_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,V,dtype", [(4096, 3000, BF16), (300, 18, F32), (6, 70001, BF16), (9, 200003, F32), (0, 5, F32), (5, 0, F32)])
def test_results_hold_no_more_than_themselves(R, V, dtype):
    """A result that is kept or saved takes its own bytes: neither the call's workspace nor the other results."""
    import ppo_amd
    if R and V:
        g, x, a = policy_inputs(R, V, dtype, R)
        batch, values = batch_of(g, x, a), torch.zeros(R, device="cuda")
    else:
        x, a, values = torch.zeros(R, V, device="cuda"), torch.zeros(R, dtype=torch.int64, device="cuda"), torch.zeros(R, device="cuda")
        batch = ppo_amd.ExperienceBatch(None, a, values, values, values, values)
    r = ppo_amd.policy_loss(x, values, batch)
    nlp, ent = ppo_amd.action_stats(x, a)
    for t, n in ((r.stats, 6), (r.dvalues, R), (r.neglogps, R), (r.entropies, R), (nlp, R), (ent, R)):
        assert t.shape == (n,) and t.dtype == F32 and t.device == x.device and t.is_contiguous() and not t.requires_grad
        assert t.untyped_storage().nbytes() == n * 4
        f = io.BytesIO()
        torch.save(t, f)
        assert f.tell() <= n * 4 + 4096                                          # the format's own records
        f.seek(0)
        assert torch.equal(torch.load(f, weights_only=True), t)


def test_results_under_the_modes_of_autograd():
    import ppo_amd
    g, x, a = policy_inputs(20, 50, F32, 1)
    b = batch_of(g, x, a)
    want, want_nlp = ppo_amd.policy_loss(x, b.new_values, b), ppo_amd.action_stats(x, a)[0]
    for mode in (torch.no_grad, torch.enable_grad, torch.inference_mode):
        with mode():
            r = ppo_amd.policy_loss(x, b.new_values, b)
            nlp, _ = ppo_amd.action_stats(x, a)
            assert r.stats.is_inference() == (mode is torch.inference_mode) and nlp.is_inference() == r.stats.is_inference()
            assert torch.equal(r.stats, want.stats) and torch.equal(nlp, want_nlp)
    nlp, _ = ppo_amd.action_stats(x, a)
    v = torch.ones(20, device="cuda", requires_grad=True)
    s = (v * nlp).sum()                                                          # saved for v's gradient
    nlp.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.backward()


def test_workspaces_are_given_back():
    """Kept results of many calls: the memory in use grows by the results, in the allocator's blocks of 512 bytes."""
    import ppo_amd
    R, V = 2048, 2100
    g, x, a = policy_inputs(R, V, BF16, 2)
    b = batch_of(g, x, a)
    out = torch.empty_like(x)
    ppo_amd.policy_loss(x, b.new_values, b, out=out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    kept = [ppo_amd.policy_loss(x, b.new_values, b, out=out).stats for _ in range(100)]
    assert torch.cuda.memory_allocated() - before == 100 * 512 and len(kept) == 100


def test_results_come_from_the_pool_that_is_in_use():
    """Memory of a captured call is the graph's own, and what a kept result holds is freed with it."""
    import ppo_amd
    g, x, a = policy_inputs(500, 2100, BF16, 3)
    b = batch_of(g, x, a)
    want = ppo_amd.policy_loss(x, b.new_values, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ppo_amd.policy_loss(x, b.new_values, b)
        nlp, ent = ppo_amd.action_stats(x, a)
    others = [torch.full((500,), 7.0, device="cuda") for _ in range(64)]         # nothing eager lands in the graph's memory
    for _ in range(3):
        for t in (r.stats, r.dvalues, r.neglogps, r.entropies, nlp, ent):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r.stats, want.stats) and torch.equal(r.neglogps, want.neglogps) and torch.equal(r.dvalues, want.dvalues)
        assert torch.equal(nlp, ppo_amd.action_stats(x, a)[0]) and all(torch.all(o == 7) for o in others)
