"""dctr_memset: any address, size and value, and as part of a captured graph, replay after replay."""
import pytest
import torch

from tf_repos_amd import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [0, 1, 255])
@pytest.mark.parametrize("at", [0, 1, 5, 15, 16])
@pytest.mark.parametrize("n", [0, 1, 3, 15, 16, 17, 31, 4095, 4096, 4097, 1000003])
def test_bytes_and_nothing_beside_them(n, at, value, dev):
    x = torch.full((at + n + 40,), 7, dtype=torch.uint8, device=dev)
    capi.check(capi.lib().dctr_memset(capi.ptr(x.data_ptr() + at), value, n, capi.current_stream()))
    want = torch.full_like(x, 7)
    want[at:at + n] = value
    assert torch.equal(x, want)


def test_more_than_the_launch_has_threads_for(dev):
    x = torch.full(((1 << 31) + 5,), 7, dtype=torch.uint8, device=dev)
    capi.check(capi.lib().dctr_memset(capi.ptr(x), 3, x.numel() - 1, capi.current_stream()))
    assert x[-1].item() == 7 and torch.all(x[:-1] == 3)


def test_replayed(dev):
    """A counter cleared and counted up by a captured graph: the same after every replay, with eager work between."""
    x = torch.zeros(8, dtype=torch.int32, device=dev)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        capi.check(capi.lib().dctr_memset(capi.ptr(x), 0, 32, capi.current_stream()))
        x.add_(5)
    for turn in range(4):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, torch.full_like(x, 5)), turn
        x.add_(turn)
        torch.cuda.synchronize()
