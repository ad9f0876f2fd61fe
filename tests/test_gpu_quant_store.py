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
