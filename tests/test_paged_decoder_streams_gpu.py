"""The decoder over the paged cache on streams of its caller."""
import pytest

torch = pytest.importorskip("torch")

from relax_b200 import ops
from test_paged_decoder_gpu import model

pytestmark = pytest.mark.gpu


def test_streams_share_no_scratch_memory(cuda_lib, monkeypatch):
    """Two sequences, each on a stream of its own, step by step: the bits of one stream, and every stream has its own counters and partial results."""
    texts = [list(range(3, 203)), list(range(400, 540))]
    steps = [(0, 150), (150, 199), (199, 200)], [(0, 100), (100, 139), (139, 140)]
    m = model()
    want = [[m.forward([s], [texts[s][a:b]]) for a, b in steps[s]] for s in (0, 1)]
    for s in (0, 1):
        m.cache.release(s)
    used = []
    of_stream = ops._stream_scratch
    monkeypatch.setattr(ops, "_stream_scratch", lambda device: used.append((torch.cuda.current_stream().cuda_stream, of_stream(device))) or used[-1][1])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    torch.cuda.synchronize()
    for i in range(3):
        for s in (0, 1):
            with torch.cuda.stream(streams[s]):
                a, b = steps[s][i]
                got[s].append(m.forward([s], [texts[s][a:b]]))
    torch.cuda.synchronize()
    for s in (0, 1):
        for x, y in zip(got[s], want[s]):
            assert torch.equal(x, y)
    memory = {stream: {t.data_ptr() for n, t in used if n == stream} for stream, _ in used}
    assert set(memory) == {s.cuda_stream for s in streams}
    assert all(len(m) == 1 for m in memory.values()) and len(set.union(*memory.values())) == 2
