"""A buffer whose rows are quantised, used from several torch streams: inserts and reads are ordered as the ordinary buffer's are,
without the caller synchronising.  A spinning kernel holds one stream back, so that a missing order shows."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
N, D, T = 64, 96, 6
SPIN = 200_000_000            # cycles: some 0.1 s


def make(seed):
    """(buffer, its T x N x D rows, the other streams of each step)."""
    import ppo_amd
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows = torch.randn(T, N, D, generator=g, device="cuda")
    acts = torch.randint(0, 9, (T, N), generator=g, device="cuda")
    rest = [torch.randn(T, N, generator=g, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    return ppo_amd.ExperienceBuffer.new_quantized(N, D, T, "int8", 32), rows, acts, rest


def insert(buf, how, rows, acts, rest):
    dones = torch.zeros_like(rest[0])
    if how == "device":
        for t in range(T):
            buf.add_experience_device(rows[t], rest[0][t], acts[t], rest[1][t], dones[t], rest[2][t])
        return
    # rows already on the device, the short streams from the host: nothing of the call waits for torch's stream
    rew, val, nlp = rest
    if how == "many":
        buf.add_many(rows, rew, acts, val, np.zeros((T, N), np.uint8), nlp)
    else:
        for t in range(T):
            buf.add_experience(rows[t], rew[t], acts[t], val[t], np.zeros(N, np.uint8), nlp[t])


def host(acts, rest):
    return acts.cpu(), [r.cpu() for r in rest]


def stored(rows):
    import ppo_amd
    s = ppo_amd.QuantizedRows(T * N, D, "int8", 32)
    s.write(rows.reshape(T * N, D))
    out = s.read()
    torch.cuda.synchronize()
    return out


def minibatches(buf, B, **kw):
    import ppo_amd
    it = ppo_amd.ExperienceBatcher(buf, B).into_iter(**kw)
    return it, it.perm().astype(np.int64)


@pytest.mark.parametrize("reader", ["pass", "training_views", "stream_view"])
@pytest.mark.parametrize("how", ["device", "step", "many"])
def test_reads_wait_for_inserts_of_another_stream(how, reader):
    buf, rows, acts, rest = make(3)
    want = stored(rows)
    insert(buf, "device", torch.zeros_like(rows), acts, rest)      # whatever is allocated once is there
    buf.returns(np.zeros(N, np.uint8))
    for _ in minibatches(buf, T * N, seed=1, bijection=True)[0]:
        pass
    torch.cuda.synchronize()
    if how != "device":
        acts, rest = host(acts, rest)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(SPIN)
        insert(buf, how, rows, acts, rest)
    with torch.cuda.stream(b):
        if reader == "training_views":
            got = buf.training_views()[0]
        elif reader == "stream_view":
            got = buf.stream_view("observations")
        else:
            buf.returns(np.zeros(N, np.uint8))
            it, perm = minibatches(buf, T * N, seed=1, bijection=True)
            got, want = next(it).observations, want[torch.from_numpy(perm).cuda()]
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    buf.close()


@pytest.mark.parametrize("streaming", [False, True])
@pytest.mark.parametrize("how", ["device", "step", "many"])
def test_inserts_wait_for_reads_of_another_stream(how, streaming):
    buf, rows, acts, rest = make(5)
    want = stored(rows)
    insert(buf, "device", rows, acts, rest)
    buf.set_streaming(streaming)
    new = torch.zeros_like(rows)
    if how != "device":
        acts, rest = host(acts, rest)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(b):
        buf.returns(np.zeros(N, np.uint8))
        it, perm = minibatches(buf, T * N, seed=1, bijection=True)
        buf.sync()
        torch.cuda._sleep(SPIN)                     # the learner is behind
        got = next(it).observations
    with torch.cuda.stream(a):
        insert(buf, how, new, acts, rest)
    torch.cuda.synchronize()
    assert torch.equal(got, want[torch.from_numpy(perm).cuda()])
    assert torch.all(buf.stream_view("observations") == 0)
    buf.close()


@pytest.mark.parametrize("reader", ["training_views", "stream_view"])
def test_inserts_wait_for_whole_reads(reader):
    buf, rows, acts, rest = make(7)
    want = stored(rows)
    insert(buf, "device", rows, acts, rest)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(b):
        torch.cuda._sleep(SPIN)
        got = buf.training_views()[0] if reader == "training_views" else buf.stream_view("observations")
    with torch.cuda.stream(a):
        insert(buf, "device", torch.zeros_like(rows), acts, rest)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    buf.close()


def test_the_same_results_as_on_one_stream():
    """Collector and learner on streams of their own, several rollouts without a host synchronisation between them."""
    results = []
    for two in (False, True):
        a = torch.cuda.Stream()
        b = torch.cuda.Stream() if two else a
        out = []
        buf, rows, acts, rest = make(9)
        for k in range(4):
            with torch.cuda.stream(a):
                torch.cuda._sleep(SPIN // 20)
                insert(buf, "device", rows * (k + 1), acts, rest)
            buf.returns(np.zeros(N, np.uint8))
            with torch.cuda.stream(b):
                it, _ = minibatches(buf, 100, seed=k)
                torch.cuda._sleep(SPIN // 20)
                out += [x.observations for x in it]
        torch.cuda.synchronize()
        results.append(out)
        buf.close()
    assert len(results[0]) == len(results[1]) and all(torch.equal(x, y) for x, y in zip(*results))


def test_a_new_buffer_is_empty_before_anything_is_inserted():
    """Its rows are set to zero on the stream that made it: inserts on another one come behind that."""
    import ppo_amd
    _, rows, acts, rest = make(11)
    want = stored(rows)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(SPIN)
        buf = ppo_amd.ExperienceBuffer.new_quantized(N, D, T, "int8", 32)
    with torch.cuda.stream(b):
        insert(buf, "device", rows, acts, rest)
        got = buf.stream_view("observations")
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(buf.training_views()[0], want)
    buf.close()


def test_a_new_pass_waits_for_reads_by_the_last_permutation():
    """A pass's permutation is overwritten by the next one only behind the reads that use it, on whichever stream they are."""
    buf, rows, acts, rest = make(13)
    want = stored(rows)
    insert(buf, "device", rows, acts, rest)
    buf.returns(np.zeros(N, np.uint8))
    for kw in (dict(bijection=True), dict(device_shuffle=True), {}):
        for seed in (1, 2):                                         # whatever is allocated once is there
            for _ in minibatches(buf, T * N, seed=seed, **kw)[0]:
                pass
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(b):
            it, perm = minibatches(buf, T * N, seed=3, **kw)
            buf.sync()
            torch.cuda._sleep(SPIN)
            got = next(it).observations
        with torch.cuda.stream(a):
            second, perm2 = minibatches(buf, T * N, seed=4, **kw)
            got2 = next(second).observations
        torch.cuda.synchronize()
        assert torch.equal(got, want[torch.from_numpy(perm).cuda()]) and torch.equal(got2, want[torch.from_numpy(perm2).cuda()])
    buf.close()


def test_sync_and_close_wait_for_rows():
    import ppo_amd
    _, rows, acts, rest = make(15)
    want = stored(rows)
    buf = ppo_amd.ExperienceBuffer.new_quantized(N, D, T, "int8", 32)
    a = torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(SPIN)
        insert(buf, "device", rows, acts, rest)
    buf.sync()
    assert torch.equal(buf.rows.read(), want)              # on the default stream, which nothing else orders
    with torch.cuda.stream(a):
        torch.cuda._sleep(SPIN)
        got = buf.stream_view("observations")
    buf.close()
    assert torch.equal(got, want)


def test_whole_reads_are_captured():
    """A read of the rows may be captured: its order with what is outside the graph is the replay's."""
    buf, rows, acts, rest = make(17)
    insert(buf, "device", rows, acts, rest)
    want = buf.stream_view("observations").clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = buf.stream_view("observations") * 2.0
    for k in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want * 2.0) and torch.equal(buf.stream_view("observations"), want)
        torch.cuda.synchronize()
    insert(buf, "device", rows * 3.0, acts, rest)
    graph.replay()
    assert torch.equal(out, stored(rows * 3.0) * 2.0)
    buf.close()
