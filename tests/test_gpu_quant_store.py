"""A QuantizedRows whose attributes were exchanged, and rows written and read in calls of every size."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def refused(store, rows):
    from ppo_amd import PpoXpPanic
    index = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: store.write(rows), lambda: store.read(), lambda: store.read(index), lambda: store.read(slice(0, 1))):
        with pytest.raises(PpoXpPanic):
            call()


def test_refuses_stores_whose_rows_overlap():
    """Exchanged tensors of the right shape whose rows share storage: expanded ones, windows that move by less than a row."""
    import ppo_amd
    x = torch.zeros(8, 64, device="cuda")
    good = ppo_amd.QuantizedRows(8, 64, "int8", 32)
    overlapping = [(good.codes[:1].expand(8, 64), good.scales), (good.codes, good.scales[:1].expand(8, 2)),
                   (torch.zeros(200, dtype=torch.int8, device="cuda").as_strided((8, 64), (16, 1)), good.scales),
                   (good.codes, torch.zeros(9, device="cuda").as_strided((8, 2), (1, 1)))]
    for codes, scales in overlapping:
        s = ppo_amd.QuantizedRows.of(good.codes, good.scales, 64, "int8", 32)
        s.codes, s.scales = codes, scales
        refused(s, x)
    # one row has no distance to the next: any stride is good
    s = ppo_amd.QuantizedRows.of(good.codes[:1], good.scales[:1], 64, "int8", 32)
    s.codes, s.scales = good.codes[:1].as_strided((1, 64), (0, 1)), good.scales[:1].as_strided((1, 2), (0, 1))
    s.write(x[:1] + 2.0)
    assert torch.all(s.read() == 2.0)


def test_refuses_a_changed_group():
    """The attributes that describe the store are looked at with each call as well."""
    import ppo_amd
    x = torch.zeros(8, 64, device="cuda")
    for name, values in (("group", (0, -1, -64, 33, 1 << 40)), ("row_size", (0, -1, 63, 1 << 40)), ("_kind", (0, 4, 3))):
        for value in values:
            s = ppo_amd.QuantizedRows(8, 64, "int8", 32)
            setattr(s, name, value)
            refused(s, x)


def test_rows_written_in_place_are_seen_by_autograd():
    """What a backward pass saved of a tensor that read or write then fills is known to be stale."""
    import ppo_amd
    store = ppo_amd.QuantizedRows(8, 64, "int8", 32)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    store.write(torch.randn(8, 64, generator=g, device="cuda"))
    index = torch.arange(4, device="cuda").int()
    w = torch.randn(64, 3, generator=g, device="cuda", requires_grad=True)
    out = torch.empty(4, 64, device="cuda")
    y = store.read(index, out=out)
    assert y is out
    loss = (y @ w).sum()                                   # saves y for the gradient of w
    store.read(index + 4, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = (store.read(index, out=out) @ w).sum()
    store.read(index + 4)                                  # a new tensor: what was saved stays good
    loss.backward()
    v = torch.randn(8, 2, generator=g, device="cuda", requires_grad=True)
    loss = (v * store.scales).sum()                        # saves the scales
    store.write(torch.ones(8, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    before = store.codes._version
    store.write(torch.ones(1, 64, device="cuda"), 3)
    assert store.codes._version > before
    with torch.inference_mode():
        out = torch.empty(4, 64, device="cuda")
        assert torch.equal(store.read(index, out=out), store.read(index))
        s = ppo_amd.QuantizedRows(8, 64, "int8", 32)
        s.write(torch.ones(8, 64, device="cuda"))


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("n", [2000, 40000])
def test_16_bit_reads_are_the_32_bit_read_rounded(n, fmt):
    """The product of a code and a scale has up to 31 significant bits: it is rounded to 32-bit numbers, and those to 16 bits, at every
    place of a row alike.  Among this many products some lie next to a border between two 16-bit numbers."""
    import ppo_amd
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    for width in (75, 64, 8):
        x = torch.randn(n, width, generator=g, device="cuda") * torch.rand(width, generator=g, device="cuda").pow(-0.5)
        store = ppo_amd.QuantizedRows(n, width, fmt, 16)
        for k in range(max(1, 200000 // n)):
            store.write(x * (1.0 + k / 64.0))
            for dtype in (torch.float16, torch.bfloat16):
                assert torch.equal(store.read(dtype=dtype), store.read().to(dtype))


# ---- calls large enough for several units a lane ------------------------------------------------------------------------------

MANY_UNITS = 256 * 256 * 4          # from here on a lane writes two units of 8 elements and reads four of 16 bytes


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,width,group", [(40000, 75, 32), (270001, 8, 16), (66001, 31, 16), (520, 4100, 32), (33000, 64, 64), (8193, 257, 256), (131073, 2, 16)])
def test_large_calls(n, width, group, dtype, fmt):
    """Ragged and even widths, apart and together, with a last workgroup that is partly filled: written, and read in order, by
    indexes of both widths and by bad ones."""
    import ppo_amd
    from test_gpu_quant_rows import code_values, quantized64, read64
    units = n * (-(-width // group) * (group // 8))
    assert units >= MANY_UNITS
    g = torch.Generator(device="cuda")
    g.manual_seed(n + width)
    wide = (torch.randn(n, width + 3, generator=g, device="cuda") * torch.rand(width + 3, generator=g, device="cuda").pow(-0.5)).to(dtype)
    wide[n // 3] = 0
    wide[n // 2, 1] = float("nan")
    q, s = quantized64(wide[:, 1:width + 1], fmt, group)
    bytes_ = (width + 1) // 2 if fmt == "int4" else width
    plain = ppo_amd.QuantizedRows(n, width, fmt, group)
    plain.write(wide[:, 1:width + 1])
    # the same rows, contiguous, into a store whose rows lie apart, behind rows of others
    kind = plain.codes.dtype
    codes, scales = torch.full((n + 5, bytes_ + 3), 9, dtype=torch.uint8, device="cuda"), torch.full((n + 5, s.shape[1] + 2), 5.0, device="cuda")
    apart = ppo_amd.QuantizedRows.of(codes.view(kind)[:, 1:bytes_ + 1], scales[:, 1:-1], width, fmt, group)
    apart.write(wide[:, 1:width + 1].contiguous(), 2)
    same = lambda x, y: torch.equal(x.nan_to_num(-7e30), y.nan_to_num(-7e30))  # noqa: E731
    assert same(plain.scales.double(), s) and torch.equal(code_values(plain), q)
    assert torch.equal(codes[2:n + 2, 1:bytes_ + 1], plain.codes.view(torch.uint8)) and same(scales[2:n + 2, 1:-1], plain.scales)
    assert torch.all(codes[:2] == 9) and torch.all(codes[n + 2:] == 9) and torch.all(codes[:, 0] == 9) and torch.all(codes[:, bytes_ + 1:] == 9)
    assert torch.all(scales[:2] == 5) and torch.all(scales[n + 2:] == 5) and torch.all(scales[:, 0] == 5) and torch.all(scales[:, -1] == 5)
    index = torch.randint(0, n, (n + 77,), generator=g, device="cuda")
    index[5], index[-1], index[-2] = -1, n + 2 ** 31 - 1 - n, n
    rows = index.clone()
    rows[(index < 0) | (index >= n)] = n - 1
    for out_t in (torch.float32, torch.bfloat16, torch.float16):
        want = read64(q, s, group, out_t)
        assert same(plain.read(dtype=out_t), want)
        out = torch.full((n, width + 5), 3.0, dtype=out_t, device="cuda")
        assert same(apart.read(slice(2, n + 2), dtype=out_t, out=out[:, 3:width + 3]), want)
        assert torch.all(out[:, :3] == 3) and torch.all(out[:, width + 3:] == 3)
        want = want[rows]
        assert same(plain.read(index, dtype=out_t), want) and same(plain.read(index.int(), dtype=out_t), want)


@pytest.fixture
def empty_cache():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def room(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB")


def test_reads_of_more_than_2_32_units(empty_cache):
    """Units are numbered in 64 bits from there on: 69 GB of output."""
    import ppo_amd
    room(80)
    store = ppo_amd.QuantizedRows(5, 64, "int8", 64)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    store.write(torch.randn(5, 64, generator=g, device="cuda"))
    each = store.read()
    n = (1 << 28) + 5                                          # 16 units a row
    index = torch.zeros(n, dtype=torch.int32, device="cuda")
    for at in (0, 1 << 14, (1 << 28) - 2, n - 5):              # the first rows, those round the 2^32nd unit, the last ones
        index[at:at + 5] = torch.tensor([1, 2, 3, 4, 2], dtype=torch.int32, device="cuda")
    out = store.read(index)
    for lo in range(0, n, 1 << 24):
        assert torch.equal(out[lo:lo + (1 << 24)], each[index[lo:lo + (1 << 24)].long()])


def test_writes_of_more_than_2_32_units(empty_cache):
    import ppo_amd
    room(110)
    n = (1 << 29) + 5                                          # 8 units a row, 69 GB of input
    x = torch.zeros(n, 64, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    places = (0, 1 << 14, (1 << 29) - 2, n - 5)
    for at in places:
        x[at:at + 5] = torch.randn(5, 64, generator=g, device="cuda").to(torch.bfloat16)
    store = ppo_amd.QuantizedRows(n, 64, "int4", 64)
    store.codes.fill_(0xff)
    store.write(x)
    left = torch.ones(n, dtype=torch.bool, device="cuda")
    for at in places:
        few = ppo_amd.QuantizedRows(5, 64, "int4", 64)
        few.write(x[at:at + 5])
        assert torch.equal(store.codes[at:at + 5], few.codes) and torch.equal(store.scales[at:at + 5], few.scales)
        left[at:at + 5] = False
    for lo in range(0, n, 1 << 26):
        here = left[lo:lo + (1 << 26)]
        assert not (store.codes[lo:lo + (1 << 26)].view(torch.int64).ne(0).any(1) & here).any() and not (store.scales[lo:lo + (1 << 26), 0].ne(0) & here).any()


def test_refused_calls_leave_no_trace():
    """What was saved of a tensor is not stale when the call that would have written it was refused."""
    import ppo_amd
    store = ppo_amd.QuantizedRows(8, 64, "int8", 32)
    out, y = torch.zeros(3, 64, device="cuda"), torch.zeros(4, 10, device="cuda")
    z, a = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    batch = ppo_amd.ExperienceBatch(None, a, z, z, z, z)
    for call in (lambda: store.write(torch.zeros(4, 64, device="cuda"), 6), lambda: store.read(slice(4, 8), out=out),
                 lambda: ppo_amd.shape_logits(y, repetition=-1.0, out=y), lambda: ppo_amd.shape_logits_backward(y, y, temperature=0.0, out=y),
                 lambda: ppo_amd.policy_loss(y, z, batch, clip=-1.0, out=y)):
        before = [t._version for t in (store.codes, store.scales, out, y)]
        with pytest.raises(ppo_amd.PpoXpPanic):
            call()
        assert [t._version for t in (store.codes, store.scales, out, y)] == before
