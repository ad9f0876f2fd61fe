"""A buffer whose rows are quantised: what its calls refuse, and what it says of itself."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
N, D, T = 4, 16, 3


def test_host_rows_of_another_layout_are_refused():
    """Arrays of the right number of elements in another order: transposed, env-major, flat, with an axis too many."""
    import ppo_amd
    buf = ppo_amd.ExperienceBuffer.new_quantized(N, D, T)
    rng = np.random.default_rng(0)
    one, many = rng.standard_normal((N, D)).astype(np.float32), rng.standard_normal((T, N, D)).astype(np.float32)
    f, ff = np.zeros(N, np.float32), np.zeros((T, N), np.float32)
    for wrap in (lambda a: a, torch.from_numpy, lambda a: torch.from_numpy(a).cuda()):
        for obs in (np.ascontiguousarray(one.T), one.reshape(-1), one[None], one.reshape(2 * N, D // 2), one.reshape(N // 2, 2 * D)):
            with pytest.raises(ppo_amd.PpoXpPanic):
                buf.add_experience(wrap(obs), f, f.astype(np.uint64), f, f.astype(np.uint8), f)
        for obs in (np.ascontiguousarray(many.transpose(1, 0, 2)), many.reshape(T * N, D), many.reshape(-1), np.ascontiguousarray(many.transpose(0, 2, 1))):
            with pytest.raises(ppo_amd.PpoXpPanic):
                buf.add_many(wrap(obs), ff, ff.astype(np.uint64), ff, ff.astype(np.uint8), ff)
    assert len(buf) == 0 and torch.all(buf.rows.codes == 0)
    buf.add_experience(one, f, f.astype(np.uint64), f, f.astype(np.uint8), f)
    buf.add_many(many[:2], ff[:2], ff[:2].astype(np.uint64), ff[:2], ff[:2].astype(np.uint8), ff[:2])
    want = ppo_amd.QuantizedRows(T * N, D)
    want.write(torch.from_numpy(np.concatenate([one[None], many[:2]]).reshape(T * N, D)).cuda())
    assert torch.equal(buf.training_views()[0], want.read())
    buf.close()


def test_its_row_size_is_its_obs_size():
    import ppo_amd
    buf = ppo_amd.ExperienceBuffer.new_quantized(N, D, T)
    assert buf.obs_size == D
    f = np.zeros(N, np.float32)
    buf.add_experience(np.zeros((N, buf.obs_size), np.float32), f, f.astype(np.uint64), f, f.astype(np.uint8), f)
    z = torch.zeros(N, device="cuda")
    buf.add_experience_device(torch.zeros(N, buf.obs_size, device="cuda"), z, z.long(), z, z, z)
    assert buf.training_views()[0].shape == (2 * N, buf.obs_size)
    buf.returns(np.zeros(N, np.uint8))
    for batch in ppo_amd.ExperienceBatcher(buf, 5):
        assert batch.observations.shape == (5, buf.obs_size)
    buf.close()
