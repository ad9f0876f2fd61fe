"""As many rows as one dispatch takes: the last of them is answered, one more is refused before anything is launched."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def zeros(rows, vocab, dtype):
    need = rows * vocab * dtype.itemsize
    if torch.cuda.mem_get_info()[0] < need + (8 << 30):
        pytest.skip(f"needs {need >> 30} GiB")
    return torch.zeros(rows, vocab, dtype=dtype, device="cuda")


@pytest.fixture(autouse=True)
def give_back():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def test_statistics_of_2_24_rows():
    import ppo_amd
    R, V = 1 << 24, 2056                                       # 69 GB
    x, a = zeros(R, V, BF16), torch.zeros(R, dtype=torch.int64, device="cuda")
    x[R - 2, 7] = 9.0
    with pytest.raises(ppo_amd.PpoXpPanic, match="too many"):
        ppo_amd.action_stats(x, a)
    nlp, ent = ppo_amd.action_stats(x[:-1], a[:-1])
    flat = nlp[:-1]
    assert torch.all(flat == flat[0]) and abs(flat[0] - math.log(V)) <= 1e-5 and torch.all(ent[:-1] == ent[0])
    assert abs(nlp[-1] - math.log(V - 1 + math.exp(9.0))) <= 1e-5


def test_rules_of_2_24_rows():
    import ppo_amd
    R, V = 1 << 24, 1032                                       # 69 GB; a row is just too long to share a workgroup
    x = zeros(R, V, F32)
    x += 1.0
    for call in (lambda: ppo_amd.shape_logits(x, temperature=0.5, out=x), lambda: ppo_amd.shape_logits_backward(x, x, temperature=0.5, out=x)):
        with pytest.raises(ppo_amd.PpoXpPanic, match="too many"):
            call()
    torch.cuda.synchronize()
    assert torch.all(x[:3] == 1) and torch.all(x[-3:] == 1)    # nothing was launched
    y = x[:-1]
    ppo_amd.shape_logits(y, temperature=0.5, out=y)
    assert all(torch.all(part == 2) for part in y.split(1 << 20)) and torch.all(x[-1] == 1)
