"""Where the token-policy operators change their route or their arithmetic could run out: many rows, offsets beyond 32 bits, several
streams at once, captured calls of every route."""
import math

import pytest
import torch

from test_gpu_policy_ops import BF16, F16, F32, U, batch_of, gen, loss64, make_rules, policy_inputs, randn, softmax64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,V,dtype", [(20000, 2100, BF16), (8193, 2049, F32), (40000, 40, F16), (70001, 5, F32), (3, 300001, BF16), (127, 66000, F16),
                                       (128, 66000, F16), (130, 140001, BF16),
                                       (260111, 65, F32), (173000, 97, F32), (168001, 100, BF16), (111200, 151, F32), (43800, 385, F32),
                                       (21900, 767, F32)])
def test_loss_routes_with_many_records(R, V, dtype):
    """Sums over several slices (more than 8192 records), workgroups that walk over rows, split rows, rows beyond the registers."""
    import ppo_amd
    g, logits, a = policy_inputs(R, V, dtype, R + V, padded=True)
    b = batch_of(g, logits, a)
    n = float((a >= 0).sum())
    r = ppo_amd.policy_loss(logits, b.new_values, b, denom=n)
    stats, stol, d, tol, dv, vtol, w = loss64(logits, b, a, float(torch.tensor(0.2)), float(torch.tensor(0.01)), 0.5, n)
    real = a >= 0
    assert torch.all(((r.neglogps.double() - w["nlp"]).abs() <= w["err_nlp"])[real])
    assert torch.all((r.dlogits.double() - d).abs() <= tol)
    assert torch.all((r.dvalues.double() - dv).abs() <= vtol)
    assert torch.all((r.stats.double() - stats).abs() <= stol + U * stats.abs())
    for _ in range(3):
        r2 = ppo_amd.policy_loss(logits, b.new_values, b, denom=n)
        assert torch.equal(r2.stats, r.stats) and torch.equal(r2.dlogits, r.dlogits)
    nlp, ent = ppo_amd.action_stats(logits, a)
    assert torch.all(((nlp.double() - w["nlp"]).abs() <= w["err_nlp"])[real]) and torch.all(((ent.double() - w["ent"]).abs() <= w["err_ent"])[real])


@pytest.mark.parametrize("R,V,dtype", [(1001, 50, F32), (1001, 63, BF16), (258200, 65, F32), (168001, 100, F16), (111200, 150, F32), (87000, 193, F32),
                                       (43700, 386, F32), (22003, 763, F32)])
def test_rows_apart_give_the_same_bits(R, V, dtype):
    """Large calls over rows that lie apart, at odd addresses: only the addresses differ, nothing beside the rows is written."""
    import ppo_amd
    g, x, a = policy_inputs(R, V, dtype, R, padded=True)
    x[5, ::2] = -math.inf
    x[6] = -math.inf
    x[7, V - 1] = math.nan
    b = batch_of(g, torch.where(torch.isfinite(x), x, 0.0), a)
    wide = torch.full((R, V + 3), 5.0, dtype=dtype, device="cuda")
    wide[:, 1:V + 1] = x
    out = torch.full((R, V + 2), 7.0, dtype=dtype, device="cuda")
    r = ppo_amd.policy_loss(x, b.new_values, b)
    q = ppo_amd.policy_loss(wide[:, 1:V + 1], b.new_values, b, out=out[:, 1:V + 1])
    same = lambda p, t: torch.equal(p.nan_to_num(1e30), t.nan_to_num(1e30))  # noqa: E731
    assert same(q.dlogits.float(), r.dlogits.float()) and same(q.neglogps, r.neglogps) and same(q.entropies, r.entropies)
    assert torch.equal(q.dvalues, r.dvalues)
    assert torch.all(out[:, 0] == 7) and torch.all(out[:, V + 1:] == 7) and torch.all(wide[:, 0] == 5) and torch.all(wide[:, V + 1:] == 5)
    pad = a < 0
    assert torch.all(r.dlogits[pad] == 0) and torch.all(r.neglogps[pad] == 0) and torch.all(r.dvalues[pad] == 0)
    if not pad[6]:
        assert torch.all(r.dlogits[6] == 0) and r.neglogps[6] == math.inf
    assert torch.all(r.dlogits[7].isnan()) if not pad[7] else torch.all(r.dlogits[7] == 0)
    if dtype == F32:          # statistics of 16-bit rows this long begin at the row's 4-byte boundary: which lane adds what follows the address
        for p, t in zip(ppo_amd.action_stats(wide[:, 1:V + 1], a), ppo_amd.action_stats(x, a)):
            assert same(p, t)


@pytest.mark.parametrize("offset,spread", [(0.0, 30.0), (80.0, 1.0), (-3000.0, 2.0), (5000.0, 2.0), (60000.0, 100.0), (-1e9, 1.0), (3e37, 1e36)])
@pytest.mark.parametrize("V", [7, 300, 5000, 150000])
def test_logits_far_from_zero(offset, spread, V):
    """A shift of all logits changes nothing but the rounding of their differences; large spreads make a row one-hot."""
    import ppo_amd
    g = gen(V)
    x = (randn(g, 12, V) * spread).double() + offset
    x = x.float()
    a = torch.randint(0, V, (12,), generator=g, device="cuda")
    a[:4] = x[:4].argmax(1)
    w = softmax64(x, a)
    nlp, ent = ppo_amd.action_stats(x, a)
    for got, want, err in ((nlp, w["nlp"], w["err_nlp"]), (ent, w["ent"], w["err_ent"])):
        big = want > 3e38                                    # beyond the range of 32 bits
        assert torch.all(((got.double() - want).abs() <= err)[~big]) and torch.all(torch.isinf(got[big]))
    b = batch_of(g, x, a)
    keep = torch.isfinite(w["nlp"]) & (w["nlp"] < 60)        # ratios of the others are 0 or 1 over numbers that no policy stores
    b.neglogps = torch.where(keep, b.neglogps, nlp)
    r = ppo_amd.policy_loss(x, b.new_values, b)
    _, _, d, tol, _, _, _ = loss64(x, b, a, float(torch.tensor(0.2)), float(torch.tensor(0.01)), 0.5, 12.0)
    over = ((r.dlogits.double() - d).abs() / tol)[keep]
    j = int(over.argmax())
    assert over.max() <= 1, (r.dlogits[keep].flatten()[j].item(), d[keep].flatten()[j].item(), tol[keep].flatten()[j].item())
    assert torch.all(torch.isfinite(r.dlogits[keep]))


def test_rows_beyond_32_bit_offsets():
    """4.4e9 elements: the last rows lie behind the 8-GiB mark of a 16-bit array."""
    import ppo_amd
    R, V = 33600, 131000
    x = torch.zeros(R, V, dtype=BF16, device="cuda")
    g = gen(3)
    x[-3:] = randn(g, 3, V).to(BF16)
    a = torch.zeros(R, dtype=torch.int64, device="cuda")
    a[-3:] = torch.tensor([1, V - 1, 77], device="cuda")
    nlp, ent = ppo_amd.action_stats(x, a)
    w = softmax64(x[-3:], a[-3:])
    assert torch.all((nlp[-3:].double() - w["nlp"]).abs() <= w["err_nlp"]) and torch.all((nlp[:-3] - math.log(V)).abs() <= 1e-5)
    hist = torch.zeros(R, 4, dtype=torch.int64, device="cuda")
    hist[-1] = torch.tensor([5, 5, V - 1, 9], device="cuda")
    before = x[-3:].clone()
    ppo_amd.shape_logits(x, history=hist, frequency=2.0, temperature=0.5, out=x)
    want = before.float()
    want[:2, 0] -= 8.0
    want[2, 5] -= 4.0
    want[2, V - 1] -= 2.0
    want[2, 9] -= 2.0
    assert torch.equal(x[-3:], (want * 2).to(BF16)) and x[0, 0] == -16 and torch.all(x[:-3, 1:] == 0)


def test_history_beyond_32_bit_offsets():
    import ppo_amd
    L = 1 << 20
    hist = torch.zeros(2100, L, dtype=torch.int32, device="cuda")            # 2.2e9 tokens
    hist[-1, -2:] = 3
    row = torch.tensor([2099, 0], dtype=torch.int32, device="cuda")
    begin = torch.tensor([L - 5, L - 1], dtype=torch.int32, device="cuda")
    out = ppo_amd.shape_logits(torch.zeros(2, 10, device="cuda"), history=hist, hist_row=row, hist_begin=begin, frequency=1.0)
    assert out[0, 0] == -3 and out[0, 3] == -2 and out[1, 0] == -1 and out[1, 3] == 0


@pytest.mark.parametrize("R,V", [(3, 70000), (5, 150000), (400, 18), (300, 700), (9000, 2100), (4, 131001)])
def test_streams_and_graphs_of_every_route(R, V):
    """The same calls on two streams at once and out of two graphs replayed side by side: nothing is shared between them."""
    import ppo_amd
    sets = []
    for seed in (1, 2):
        g, x, a = policy_inputs(R, V, BF16, seed)
        b = batch_of(g, x, a)
        kw = make_rules(g, R, V, 40, "bits", "none", "rows")
        sets.append((x, a, b, kw, torch.randn(200, 96, generator=g, device="cuda"), torch.randperm(200, generator=g, device="cuda").int()))
    stores = [ppo_amd.QuantizedRows(200, 96, "int8", 32) for _ in sets]

    def work(k):
        x, a, b, kw, rows, idx = sets[k]
        y = ppo_amd.shape_logits(x, **kw)
        n, h = ppo_amd.action_stats(x, a)
        r = ppo_amd.policy_loss(x, b.new_values, b)
        bk = {q: v for q, v in kw.items() if q not in ("bias", "presence", "frequency", "gen_begin")}
        d = ppo_amd.shape_logits_backward(r.dlogits, x, **bk)
        stores[k].write(rows)
        return [y, n, h, r.stats, r.dlogits, r.dvalues, d, stores[k].read(idx)]
    want = [[t.clone() for t in work(k)] for k in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got.append(work(k))
        torch.cuda.synchronize()
        for k in (0, 1):
            for t, u in zip(got[k], want[k]):
                assert torch.equal(t.float().nan_to_num(1), u.float().nan_to_num(1))
    graphs, outs = [], []
    for k in (0, 1):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(work(k))
        graphs.append(gr)
    for _ in range(3):
        for k in (0, 1):
            for t in outs[k]:
                t.zero_()
        torch.cuda.synchronize()
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        eager = work(0)
        torch.cuda.synchronize()
        for k in (0, 1):
            for t, u in zip(outs[k], want[k]):
                assert torch.equal(t.float().nan_to_num(1), u.float().nan_to_num(1))
        assert torch.equal(eager[4], want[0][4])


def test_current_device_and_autograd_state_are_left_alone():
    import ppo_amd
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    y = ppo_amd.shape_logits(x, temperature=2.0)
    assert not y.requires_grad and torch.equal(y, x.detach() * 0.5)
    a = torch.zeros(3, dtype=torch.int64, device="cuda")
    n, _ = ppo_amd.action_stats(x, a)
    assert not n.requires_grad and torch.cuda.current_device() == 0
    # gradients are handed on by the caller
    d = ppo_amd.shape_logits_backward(torch.ones(3, 50, device="cuda"), x, temperature=2.0)
    x.backward(d)
    assert torch.all(x.grad == 0.5)


def test_threads_call_at_once():
    """Calls release the interpreter while they launch: each thread on a stream of its own gets what it gets alone."""
    import threading
    import ppo_amd
    shapes = [(300, 18, F32), (64, 700, BF16), (4, 70001, F16), (3, 150000, F32)]
    jobs, wrong = [], []
    for k, (R, V, dtype) in enumerate(shapes):
        g, x, a = policy_inputs(R, V, dtype, 100 + k)
        b = batch_of(g, x, a)
        hist = torch.randint(0, V, (R, 33), generator=g, device="cuda")
        store = ppo_amd.QuantizedRows(R, 70, "int8", 32)
        rows = randn(g, R, 70)

        def work(x=x, a=a, b=b, hist=hist, store=store, rows=rows):
            y = ppo_amd.shape_logits(x, history=hist, repetition=1.3, frequency=0.1)
            store.write(rows)
            r = ppo_amd.policy_loss(y, b.new_values, b)
            d = ppo_amd.shape_logits_backward(r.dlogits, x, history=hist, repetition=1.3)
            return [y, *ppo_amd.action_stats(y, a), r.stats, r.dvalues, d, store.read()]
        jobs.append((work, work()))
    torch.cuda.synchronize()

    def run(work, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got = [work() for _ in range(30)]
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(p, q) for out in got for p, q in zip(out, want)):
                    wrong.append("results differ")
                try:
                    ppo_amd.shape_logits(want[0], repetition=-1.0)
                    wrong.append("not refused")
                except ppo_amd.PpoXpPanic as e:
                    if "repetition" not in str(e):
                        wrong.append(str(e))
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))
    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
