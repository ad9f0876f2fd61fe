"""Row stores refuse what does not describe one before their tensors are looked at.  Runs without a GPU."""
import pytest
import torch

from ppo_amd import PpoXpPanic, _lib


@pytest.mark.parametrize("group", [0, -1, -64])
def test_group_must_be_positive(group):
    T = _lib.torchcall()
    codes, scales, x = torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8, 2), torch.zeros(8, 64)
    for call in (lambda: T.write(codes, scales, 64, 1, group, x, 0), lambda: T.read(codes, scales, 64, 1, group, None, 0, 8, 0, None)):
        with pytest.raises(PpoXpPanic, match=f"group {group} "):
            call()
