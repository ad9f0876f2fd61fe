"""QuantizedRows against the formats' definitions evaluated in 64 bits: codes, scales and read values are equal, not close (the
stored scale and the read value are one rounding each of a 64-bit value, the code is the exactly nearest one)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOP = {"int8": 127, "int4": 7, "e4m3": 448}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def quantized64(rows, fmt, group):
    """(code values [n, width] f64, scales [n, groups] f64)."""
    n, width = rows.shape
    G = -(-width // group)
    x = torch.nn.functional.pad(rows.double(), (0, G * group - width)).reshape(n, G, group)
    top = x.abs().amax(2)
    bad = ~torch.isfinite(x).all(2)
    if fmt == "e4m3":
        k = torch.ceil(torch.log2(top / 448) - 1e-12)
        s = torch.exp2(k)
    else:
        s = (top / TOP[fmt]).float().double()
    s = torch.where(top < 2.0 ** -110, 0.0, s)
    q = torch.where(s[..., None] > 0, x / s[..., None], 0.0)
    if fmt == "e4m3":
        unit = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
        q = torch.round(q / unit) * unit
    else:
        q = torch.round(q)
    s = torch.where(bad, math.nan, s)
    q = torch.where(bad[..., None], 0.0, q)
    return q.reshape(n, -1)[:, :width], s


def code_values(store):
    if store.format == "int8":
        return store.codes.double()
    if store.format == "e4m3":
        return store.codes.float().double()
    b = store.codes.view(torch.int8).int()
    lo, hi = ((b & 15) ^ 8) - 8, b >> 4
    return torch.stack((lo, hi), 2).reshape(b.shape[0], -1)[:, :store.row_size].double()


def read64(q, s, group, dtype):
    wide = s.repeat_interleave(group, 1)[:, :q.shape[1]]
    return (q * wide).float().to(dtype) if dtype != F32 else (q * wide).float()   # the product of 8 and 24 bits fits 32 exactly


CASES = [(1, 1, 16), (3, 5, 32), (2, 16, 16), (7, 17, 16), (5, 31, 32), (4, 33, 32), (300, 64, 64), (65, 100, 64), (9, 128, 128), (6, 257, 256),
         (3, 1000, 512), (2, 4100, 32), (1, 8191, 64), (1025, 8, 16)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,width,group", CASES)
def test_write_and_read(n, width, group, dtype, fmt):
    import ppo_amd
    g = gen(n * 7 + width)
    x = torch.randn(n, width, generator=g, device="cuda") * torch.rand(width, generator=g, device="cuda").pow(-0.5)
    if n > 2:
        x[1] = 0
        x[2] *= 1e-4
    x = x.to(dtype)
    q, s = quantized64(x, fmt, group)
    store = ppo_amd.QuantizedRows(n + 3, width, fmt, group)
    store.write(x, 2)
    assert torch.equal(code_values(store)[2:n + 2], q) and torch.equal(store.scales[2:n + 2].double(), s)
    for k in (0, 1, n + 2):                                                     # the rows beside them stay zero
        assert torch.all(store.codes.view(torch.uint8)[k] == 0) and torch.all(store.scales[k] == 0)
    for out_t in (F32, BF16, F16):
        want = read64(q, s, group, out_t)
        assert torch.equal(store.read(slice(2, n + 2), dtype=out_t), want)
        idx = torch.randint(0, n, (2 * n + 5,), generator=g, device="cuda")
        assert torch.equal(store.read((idx + 2).int(), dtype=out_t), want[idx])
        assert torch.equal(store.read(idx + 2, dtype=out_t), want[idx])
    assert torch.equal(store.read()[2:n + 2], read64(q, s, group, F32)) and len(store.read()) == n + 3


@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_ties_and_borders_round_exactly(fmt):
    """Quotients that are ties, and one step to either side of a tie, for scales whose reciprocal is not exact."""
    import ppo_amd
    top = TOP[fmt]
    rows = []
    for s in (1.0, 1.1, 0.3, 7.7e-5, 3.3e12, 1.9999999):
        s = torch.tensor(s, dtype=F32)
        amax = (s.double() * top).float()
        s = (amax.double() / top).float()
        tie = (torch.arange(-top, top, device="cpu").double() + 0.5) * s.double()
        v = tie.float()
        row = torch.cat([amax[None], v, torch.nextafter(v, v * 0), torch.nextafter(v, v * 4), -v])
        row = torch.where(row.abs() > amax, amax, row)
        rows.append(row)
    x = torch.stack(rows).cuda()
    width = x.shape[1]
    group = 512
    # one group per row that holds the maximum: pieces of 511 values behind it
    pieces = [torch.cat([x[:, :1], x[:, 1 + k:1 + k + 511]], 1) for k in range(0, width - 1, 511)]
    for p in pieces:
        q, s = quantized64(p, fmt, group)
        store = ppo_amd.QuantizedRows(p.shape[0], p.shape[1], fmt, group)
        store.write(p.contiguous())
        assert torch.equal(store.scales.double(), s) and torch.equal(code_values(store), q)


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_extremes(fmt, dtype):
    import ppo_amd
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.zeros(8, 64, device="cuda")
    x[0, 3], x[0, 40] = math.nan, 1.0                                           # groups of 32: the other one is untouched
    x[1, 33], x[1, 0] = math.inf, 2.0
    x[2, 0], x[2, 1], x[2, 40] = big, -big, tiny
    x[3, 0] = 2.0 ** -111 if dtype != F16 else 2.0 ** -24
    x[4, :] = -0.0
    x[5, 0], x[5, 1] = 1.0, 1e-30
    x[6, 0] = 2.0 ** -110 if dtype != F16 else 2.0 ** -23
    x[7, 0], x[7, 1], x[7, 2] = 448.0, 0.001, -449.0
    x = x.to(dtype)
    q, s = quantized64(x, fmt, 32)
    store = ppo_amd.QuantizedRows(8, 64, fmt, 32)
    store.write(x)
    assert torch.equal(store.scales.double().nan_to_num(-5), s.nan_to_num(-5)) and torch.equal(code_values(store), q)
    back = store.read()
    assert torch.all(back[0, :32].isnan()) and torch.all(back[1, 32:].isnan())
    assert not back[0, 32:].isnan().any() and not back[1, :32].isnan().any() and not back[2:].isnan().any()


def test_error_is_at_most_half_a_step():
    import ppo_amd
    x = torch.randn(1000, 96, generator=gen(2), device="cuda")
    for fmt in ("int8", "int4"):
        store = ppo_amd.QuantizedRows(1000, 96, fmt, 32)
        store.write(x)
        step = store.scales.repeat_interleave(32, 1)
        assert torch.all((store.read() - x).abs() <= step * (0.5 + 2.0 ** -16))
    store = ppo_amd.QuantizedRows(1000, 96, "e4m3", 32)
    store.write(x)
    step = store.scales.repeat_interleave(32, 1)
    assert torch.all((store.read() - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, step * 2.0 ** -10))


def test_strides_and_bad_indexes():
    import ppo_amd
    g = gen(4)
    n, width = 40, 75
    wide = torch.randn(n, width + 6, generator=g, device="cuda")
    x = wide[:, 3:3 + width]
    codes = torch.full((n + 2, width + 5), 9, dtype=torch.int8, device="cuda")
    scales = torch.full((n + 2, 9), 5.0, device="cuda")
    store = ppo_amd.QuantizedRows.of(codes[:, 1:1 + width], scales[:, 2:5], width, "int8", 32)
    store.write(x, 1)
    q, s = quantized64(x, "int8", 32)
    assert torch.equal(codes[1:n + 1, 1:1 + width].double(), q) and torch.equal(scales[1:n + 1, 2:5].double(), s)
    edge = torch.ones_like(codes, dtype=torch.bool)
    edge[1:n + 1, 1:1 + width] = False
    assert torch.all(codes[edge] == 9)
    out = torch.full((6, width + 4), 3.0, dtype=BF16, device="cuda")
    idx = torch.tensor([0, 5, -1, n + 1, n + 2, 2 ** 31 - 1], device="cuda")
    got = store.read(idx, dtype=BF16, out=out[:, 2:2 + width])
    last = store.read(slice(n + 1, n + 2), dtype=BF16)[0]
    for k in range(2, 6):
        assert torch.equal(got[k], last)                                        # outside the store: the last row
    assert torch.equal(got[1], store.read(slice(5, 6), dtype=BF16)[0])
    assert torch.all(out[:, :2] == 3) and torch.all(out[:, 2 + width:] == 3)
    assert torch.equal(store.read(idx.int(), dtype=BF16), got)
    assert store.read(idx[:0]).shape == (0, width) and store.read(slice(3, 3)).shape == (0, width)


def test_store_beyond_32_bit_offsets():
    """Rows behind the 4-GiB mark of the codes."""
    import ppo_amd
    width, n = 1 << 16, (1 << 16) + 40
    store = ppo_amd.QuantizedRows(n, width, "int8", 512)
    x = torch.randn(5, width, generator=gen(6), device="cuda")
    store.write(x, n - 5)
    q, s = quantized64(x, "int8", 512)
    assert torch.equal(store.codes[n - 5:].double(), q)
    idx = torch.tensor([n - 1, 0, n - 5], device="cuda", dtype=torch.int32)
    got = store.read(idx)
    want = read64(q, s, 512, F32)
    assert torch.equal(got[0], want[4]) and torch.all(got[1] == 0) and torch.equal(got[2], want[0])


def test_captured_and_replayed():
    import ppo_amd
    g = gen(9)
    x = torch.randn(100, 130, generator=g, device="cuda", dtype=F32)
    idx = torch.randperm(100, generator=g, device="cuda").int()
    store = ppo_amd.QuantizedRows(100, 130, "int4", 32)
    store.write(x)
    want = store.read(idx)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        store.write(x)
        out = store.read(idx)
    for k in range(3):
        store.codes.zero_()
        out.zero_()
        gr.replay()
        assert torch.equal(out, want)
        assert torch.equal(store.read(idx), want)
        torch.cuda.synchronize()


def test_refusals():
    import ppo_amd
    from ppo_amd import PpoXpPanic
    store = ppo_amd.QuantizedRows(8, 64, "int8", 64)
    x = torch.zeros(4, 64, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    for call in (lambda: store.write(x, 5), lambda: store.write(x, -1), lambda: store.write(x[:, :63]), lambda: store.write(x.double()),
                 lambda: store.write(x.cpu()), lambda: store.write(x.t()), lambda: store.read(i.short()), lambda: store.read(i.cpu()),
                 lambda: store.read(i[None]), lambda: store.read(slice(0, 8, 2)), lambda: store.read(i, dtype=torch.float64),
                 lambda: store.read(i, out=x), lambda: store.read(i, dtype=BF16, out=x[:3]),
                 lambda: ppo_amd.QuantizedRows.of(store.codes, store.scales, 64, "int4", 64),
                 lambda: ppo_amd.QuantizedRows.of(store.codes, store.scales[:, :0], 64, "int8", 64),
                 lambda: ppo_amd.QuantizedRows(4, 64, "int8", 48).write(x)):
        with pytest.raises(PpoXpPanic):
            call()
    with pytest.raises(PpoXpPanic):
        ppo_amd.QuantizedRows(0, 64).read(i)


def test_refuses_tensors_that_no_longer_fit():
    """codes and scales are attributes: exchanged ones are looked at before they are used."""
    import ppo_amd
    from ppo_amd import PpoXpPanic
    x = torch.zeros(8, 64, device="cuda")
    good = ppo_amd.QuantizedRows(8, 64, "int8", 32)
    for codes, scales in ((good.codes[:4], good.scales), (good.codes, good.scales[:4]), (good.codes[:, :63], good.scales), (good.codes, good.scales[:, :1]),
                          (good.codes.cpu(), good.scales), (good.codes, good.scales.cpu()), (good.codes.int(), good.scales), (good.codes, good.scales.double()),
                          (good.codes.t().contiguous().t(), good.scales), (good.codes[0], good.scales)):
        s = ppo_amd.QuantizedRows.of(good.codes, good.scales, 64, "int8", 32)
        s.codes, s.scales = codes, scales
        for call in (lambda: s.write(x), lambda: s.read()):
            with pytest.raises(PpoXpPanic):
                call()
    s = ppo_amd.QuantizedRows(8, 64, "int8", 32)
    s.codes, s.scales = torch.ones_like(good.codes), torch.full_like(good.scales, 2.0)      # others of the same shapes are the store now
    assert torch.all(s.read() == 2.0)
