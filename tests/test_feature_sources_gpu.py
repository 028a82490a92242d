"""Stores encoded from CUDA tensors: the tensor's stream and device are the caller's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "i8", "f8"])
def test_rows_written_on_another_stream(dtype):
    """Rows that a side stream is still writing when the store is made in it."""
    from aethergraph_b200 import FeatureStore

    n, dim = 20_000, 64
    final = torch.randint(-64, 65, (n, dim), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).float()
    ids = torch.arange(n, device="cuda")
    want = FeatureStore.from_array(final.cpu().numpy(), dtype).gather(ids)
    x = torch.zeros(n, dim, device="cuda")
    a = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):  # about 100 ms of work before the rows are written
            a = a @ a
            a = a / a.abs().max()
        x.copy_(final)
        store = FeatureStore.from_array(x, dtype)
        x.zero_()  # the store holds rows of its own
        got = store.gather(ids)
    side.synchronize()
    assert torch.equal(got, want)


def test_the_store_is_on_the_tensors_device():
    from aethergraph_b200 import FeatureStore

    x = torch.ones(4, 8, device="cuda")
    assert FeatureStore.from_array(x)._device == x.get_device()
    assert FeatureStore.from_array(x, device=x.get_device())._device == x.get_device()
    with pytest.raises(ValueError, match="cuda:"):
        FeatureStore.from_array(x, "f8", device=x.get_device() + 1)
