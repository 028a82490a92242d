"""Whose error it is: ids outside a store's rows are reported by that store, others by the device's check."""
import threading

import pytest
import torch

from test_ops_gpu import ops, product_case, rand  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture()
def stores(ops):  # noqa: F811
    from aethergraph_b200 import FeatureStore

    return [FeatureStore.from_f8(*ops.encode_f8(rand(i, 20, 64))) for i in range(2)], ops.encode_weight_f8(rand(9, 48, 64))


@pytest.mark.parametrize("rows", [2, 300])  # both kernels
def test_a_stores_products_are_its_own(ops, stores, rows):  # noqa: F811
    (a, b), w = stores
    bad = torch.zeros(rows, dtype=torch.int64, device="cuda")
    bad[1] = 20
    out = a.project(bad, *w)
    b.check()
    ops.check()
    with pytest.raises(ValueError, match="out of bounds"):
        a.check()
    a.check()
    assert not bool(out[1].any()) and bool(out[0].any())
    case = product_case(20, 64, 48)
    ops.product_f8(*case, ids=bad)
    a.check()
    b.check()
    with pytest.raises(ValueError, match="out of bounds"):
        ops.check()
    ops.check()


def test_gather_and_product_of_one_store(ops, stores):  # noqa: F811
    """One report for what came before it, and none left over for another's check."""
    (a, b), w = stores
    bad = torch.tensor([0, 99], device="cuda")
    a.gather(bad)
    a.project(bad, *w)
    with pytest.raises(ValueError, match="out of bounds"):
        a.check()
    a.check()
    b.check()
    ops.check()


def test_threads(ops, stores):  # noqa: F811
    """A thread with bad ids and one without, each on a stream of its own."""
    pair, w = stores
    told = [0, 0]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            ids = torch.full((200,), 25 if i else 3, device="cuda")
            for _ in range(20):
                pair[i].project(ids, *w)
                try:
                    pair[i].check()
                except ValueError:
                    told[i] += 1

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert told == [0, 20]


def test_a_store_in_other_types_has_no_product(ops):  # noqa: F811
    from aethergraph_b200 import FeatureStore

    ids = torch.zeros(2, dtype=torch.int64, device="cuda")
    for dtype in ("f32", "bf16", "i8"):
        with pytest.raises(ValueError, match="8-bit float rows"):
            FeatureStore.from_array(rand(1, 4, 64), dtype).project(ids, *ops.encode_weight_f8(rand(2, 8, 64)))


@pytest.mark.parametrize("dtype", ["f32", "f8"])
def test_a_store_that_goes_while_it_is_read(ops, dtype):  # noqa: F811
    """The last reference to a store goes right after its calls, which wait behind other work."""
    from aethergraph_b200 import FeatureStore

    x = rand(1, 50_000, 128)
    ids = torch.randint(0, 50_000, (100_000,), device="cuda")
    w = ops.encode_weight_f8(rand(2, 64, 128))
    kept = FeatureStore.from_array(x, dtype)
    want = kept.gather(ids), kept.project(ids, *w) if dtype == "f8" else None
    a = torch.randn(4096, 4096, device="cuda")
    for _ in range(3):
        store = FeatureStore.from_array(x, dtype)
        for _ in range(30):
            a = a @ a
            a = a / a.abs().max()
        got = store.gather(ids), store.project(ids, *w) if dtype == "f8" else None
        del store
        assert torch.equal(got[0], want[0]) and (dtype != "f8" or torch.equal(got[1], want[1]))


def test_where_a_stores_rows_are(ops, stores):  # noqa: F811
    """The rows of a store, for a product of the C ABI without the store."""
    import ctypes as C

    from aethergraph_b200 import FeatureStore, _lib

    codes, scales = ops.encode_f8(rand(1, 6, 40))
    store = FeatureStore.from_f8(codes, scales)
    at, s, pitch = C.c_void_p(), C.c_void_p(), C.c_uint64()
    _lib.check(_lib.lib().ag_features_f8_rows(store._h, C.byref(at), C.byref(s), C.byref(pitch)))
    assert (at.value, s.value, pitch.value) == (codes.data_ptr(), scales.data_ptr(), codes.stride(0))
