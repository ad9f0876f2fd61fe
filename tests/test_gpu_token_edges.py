"""Arguments of the logit rules and the objective at the ends of their types' ranges."""
import pytest
import torch

from test_gpu_policy_ops import BF16, F16, F32, batch_of, check_shape, gen, half, policy_inputs, randn, rules64

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LAST, FIRST = 2 ** 31 - 1, -2 ** 31

# short rows that share a workgroup, a workgroup a row with few and with many chunks; histories short and long for their vocabulary
ROUTES = [(12, 50, 40), (12, 50, 2), (12, 5000, 40), (12, 5000, 700), (96, 20011, 40), (96, 20011, 900), (520, 3000, 90)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V,L", ROUTES)
def test_history_positions_at_the_ends_of_32_bits(R, V, L, dtype):
    """Positions are clamped to the history: a begin far behind it leaves nothing, an end far behind it all of it."""
    import ppo_amd
    g = gen(R + V + L)
    x = (randn(g, R, V) * 2).to(dtype)
    hist = torch.randint(0, V, (R, L), generator=g, device="cuda")
    i32 = lambda *v: torch.tensor([v[k % len(v)] for k in range(R)], dtype=torch.int64, device="cuda").int()  # noqa: E731
    kw = dict(history=hist, repetition=1.5, presence=0.25, frequency=0.5, temperature=0.75,
              hist_begin=i32(LAST, 0, FIRST, LAST - 255, L, LAST - 1, L - 1, 1),
              hist_end=i32(LAST, L, LAST, L + 1, FIRST, 0, LAST - 3),
              gen_begin=i32(0, LAST, FIRST, L, LAST - 7))
    check_shape(x, ppo_amd.shape_logits(x, **kw), kw)
    grad = randn(g, R, V).to(dtype)
    bk = {k: v for k, v in kw.items() if k not in ("presence", "frequency", "gen_begin")}
    got = ppo_amd.shape_logits_backward(grad, x, **bk).cpu().double()
    seen, _, _, rep, _, _, temp = rules64(x, kw, V)
    d = grad.cpu().double()
    want = torch.where(seen, torch.where(x.cpu().double() > 0, d / rep, d * rep), d) / temp
    # 1 / T, 1 / rep, their product and the product with it, then the rounding to the type
    assert torch.all((got - want).abs() <= (half(dtype) + 4 * U) * want.abs() * (1 + half(dtype)) + 2.0 ** -25 * (dtype == F16))


@pytest.mark.parametrize("R,V,L", ROUTES)
def test_divisors_at_the_ends_of_their_range(R, V, L):
    """The least and the largest scalars, and rows whose own value lies below the least: those count as the least one."""
    import ppo_amd
    g = gen(R + V)
    x = randn(g, R, V)
    x[:, ::5] = 0.0                                            # 0 divided by anything is 0
    x[:, 1::5] *= 2.0 ** -100
    hist = torch.randint(0, V, (R, L), generator=g, device="cuda")
    least, most = 2.0 ** -126, float(torch.finfo(F32).max)
    grad = x.flip(0) * 2.0 ** -30
    for kw in (dict(temperature=least), dict(repetition=least), dict(temperature=least, repetition=most), dict(temperature=2.0 ** 126), dict(repetition=2.0 ** 126)):
        kw["history"] = hist
        seen, _, _, rep, _, _, temp = rules64(x, kw, V)
        d, l = grad.cpu().double(), x.cpu().double()
        got, want = ppo_amd.shape_logits(x, **kw).cpu().double(), torch.where(seen, torch.where(l > 0, l / rep, l * rep), l) / temp
        # The reciprocal of a divisor above 2^126 is a multiple of 2^-149 and at least 2^-128: off by 2^-150 / 2^-128 = 4 u.  Two of
        # them, two products: 10 u.  A quotient below 2^-126 in between is a multiple of 2^-149 as well, off by 2^-150, which the
        # division by the temperature magnifies.
        fits = want.abs() < 2.0 ** 127
        assert torch.all(((got - want).abs() <= 10 * U * want.abs() + 2.0 ** -150 / temp.clamp(max=1.0) + 2.0 ** -150)[fits]) and not got.isnan().any()
        slope = torch.where(seen, torch.where(l > 0, 1 / rep, rep), 1.0) / temp
        got, want = ppo_amd.shape_logits_backward(grad, x, **kw).cpu().double(), d * slope
        # the slope is one 32-bit number, the product of two reciprocals or of one and the repetition: 4 u + 4 u + u, and the product
        # with the gradient
        inside = (slope.abs() < 2.0 ** 127) & (want.abs() < 2.0 ** 127) & (slope.abs() >= 2.0 ** -126)
        assert torch.all(((got - want).abs() <= 10 * U * want.abs() + 2.0 ** -149)[inside]) and not got[inside].isnan().any()
    f = lambda *v: torch.tensor([v[k % len(v)] for k in range(R)], dtype=F32, device="cuda")  # noqa: E731
    below, held = f(0.0, -1.0, 2.0 ** -149, 2.0 ** -128, 2.0 ** -126, 1.0), f(least, least, least, least, least, 1.0)
    for name in ("temperature", "repetition"):
        got, want = (ppo_amd.shape_logits(x, history=hist, **{name: v}) for v in (below, held))
        assert torch.equal(got, want) and not got.isnan().any()
        got, want = (ppo_amd.shape_logits_backward(grad, x, history=hist, **{name: v}) for v in (below, held))
        assert torch.equal(got, want) and not got.isnan().any()
    bad = f(float("nan"), 1.0)
    got = ppo_amd.shape_logits(x, temperature=bad)
    assert got[::2].isnan().all() and torch.equal(got[1::2], x[1::2])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V,L", ROUTES)
def test_an_infinite_penalty_forbids_the_tokens_it_applies_to(R, V, L, dtype):
    import ppo_amd
    g = gen(V)
    x = randn(g, R, V).to(dtype)
    hist = torch.randint(0, V, (R, L), generator=g, device="cuda")
    half_way = torch.full((R,), L // 2, dtype=torch.int32, device="cuda")
    counted = torch.zeros(R, V, device="cuda").scatter_(1, hist[:, L // 2:], 1.0) > 0      # tokens of the prompt only are not counted
    inf = torch.full((R,), float("inf"), device="cuda")
    inf[::3] = 0.0
    for kw in (dict(frequency=inf), dict(presence=inf), dict(frequency=inf, presence=inf)):
        out = ppo_amd.shape_logits(x, history=hist, gen_begin=half_way, **kw)
        forbidden = counted & (inf > 0)[:, None]
        assert torch.all(out[forbidden] == -float("inf")) and torch.equal(out[~forbidden], x[~forbidden])


@pytest.mark.parametrize("R,V", [(200, 18), (70, 151), (40, 5000), (6, 70001), (300, 20011)])
def test_the_denominator_scales_what_is_over_it(R, V):
    """rows / S with a power of two: statistics and gradients are S times as large to the last bit."""
    import ppo_amd
    g, x, a = policy_inputs(R, V, F32, R + V)
    b = batch_of(g, x, a)
    S = 2.0 ** 16
    r, q = (ppo_amd.policy_loss(x, b.new_values, b, denom=n) for n in (float(R), R / S))
    assert torch.equal(q.stats, r.stats * S) and torch.equal(q.dvalues, r.dvalues * S)
    assert torch.equal(q.neglogps, r.neglogps) and torch.equal(q.entropies, r.entropies)
    normal = r.dlogits.abs() >= 2.0 ** -100                    # a factor below 2^-126 has fewer bits, and its product with S keeps them
    assert torch.equal(q.dlogits[normal], r.dlogits[normal] * S) and torch.all(q.dlogits[~normal].abs() <= 2.0 ** -83)


def test_f16_gradients_that_only_a_scale_keeps():
    import ppo_amd
    R, V, S = 2048, 30011, 2.0 ** 16
    g, x, a = policy_inputs(R, V, F16, 5)
    b = batch_of(g, x, a)
    want = ppo_amd.policy_loss(x.float(), b.new_values, b).dlogits
    plain = ppo_amd.policy_loss(x, b.new_values, b).dlogits
    assert (plain == 0).float().mean() > 0.5                   # what the documentation warns of
    got = ppo_amd.policy_loss(x, b.new_values, b, denom=R / S).dlogits.float() / S
    # the same statistics in 32 bits by another route (V / 1000 and 48 additions, as many powers of 2 u, 25 |d| u at most), one rounding to
    # f16, half of its least subnormal over S
    size = want.abs() * (half(F16) + 400 * U) + 2.0 ** -25 / S
    p = torch.softmax(x.float(), 1)
    ent = 0.01 * p * 40 * 400 * U / R                          # where ln p + H cancels: both below 20 here
    assert torch.all((got - want).abs() <= size + ent)
