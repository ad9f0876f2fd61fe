"""Row stores refuse what does not describe one before their tensors are looked at.  Runs without a GPU."""
import pytest
import torch

from ppo_amd import ExperienceBuffer, PpoXpPanic, QuantizedRows, _lib


@pytest.mark.parametrize("group", [0, -1, -64])
def test_group_must_be_positive(group):
    T = _lib.torchcall()
    codes, scales, x = torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8, 2), torch.zeros(8, 64)
    for call in (lambda: T.write(codes, scales, 64, 1, group, x, 0), lambda: T.read(codes, scales, 64, 1, group, None, 0, 8, 0, None)):
        with pytest.raises(PpoXpPanic, match=f"group {group} "):
            call()


@pytest.mark.parametrize("what,bad", [("format", "int2"), ("format", None), ("group", 0), ("group", 8), ("group", 48), ("group", 1024), ("group", -64),
                                      ("row_size", 0), ("row_size", -1), ("row_size", (1 << 24) + 1)])
def test_what_no_call_could_use_is_refused_when_it_is_made(what, bad):
    kw = {"row_size": 64, "format": "int8", "group": 64, what: bad}
    codes, scales = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1)
    for call in (lambda: QuantizedRows(4, **kw), lambda: QuantizedRows.of(codes, scales, **kw),
                 lambda: ExperienceBuffer.new_quantized(4, kw["row_size"], 3, kw["format"], kw["group"])):
        with pytest.raises(PpoXpPanic):
            call()


@pytest.mark.parametrize("dtype", [torch.float64, torch.int8, torch.float8_e4m3fn])
def test_a_buffer_whose_rows_could_not_be_read_is_not_made(dtype):
    with pytest.raises(PpoXpPanic, match="f32, bf16 or f16"):
        ExperienceBuffer.new_quantized(4, 64, 3, dtype=dtype)
