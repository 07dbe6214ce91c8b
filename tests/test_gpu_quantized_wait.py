"""Scans whose waits run out: reported, and nothing that was not made is given back as a result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def status():
    from vectorlink_gpu import _lib
    return _lib.read_status(torch.device(DEV))


def scan(store, q, metric, out):
    if metric == "product":
        return store.product(q, rows=(1, len(store)), out=out)
    return store.distances(q, rows=(1, len(store)), metric=metric, out=out)


# Rows of 131,072 columns: a tile takes a thousand copies, far longer than a microsecond.  40,000 queries are several blocks for a CTA.
# The last three may or may not run out.
@pytest.mark.parametrize("count,dim,nq,surely", [(2001, 131072, 1, True), (2001, 131072, 300, True), (1000, 131072, 20, True), (301, 16384, 40_000, True), (40_001, 96, 100, False),
                                                 (40_001, 96, 7, False), (30_001, 1024, 600, False)])
@pytest.mark.parametrize("metric,dtype,pad", [("l2", torch.float32, 0), ("cosine", torch.float32, 3), ("product", torch.bfloat16, 1), ("product", torch.float16, 0)])
def test_results_that_were_not_made_are_no_numbers(count, dim, nq, surely, metric, dtype, pad):
    from vectorlink_gpu import QuantizedVectors
    g = torch.Generator(device=DEV).manual_seed(count + nq)
    store = QuantizedVectors(count, dim, device=DEV)
    for lo in range(0, count, 500):
        store.write(torch.randn((min(500, count - lo), dim), generator=g, device=DEV), first_row=lo)
    q = torch.randn((nq, dim), generator=g, device=DEV)

    def result():
        return torch.full((nq, count - 1 + pad), 7.0, dtype=dtype, device=DEV)

    want, got, after = result(), result(), result()
    status()
    scan(store, q, metric, want[:, :count - 1])
    assert status() == 0 and not want.isnan().any()
    store.wait_us = 1
    scan(store, q, metric, got[:, :count - 1])
    found = status()
    assert found in (0, 4) and (found == 4 or not surely)
    missing = got.isnan()
    assert torch.equal(got[~missing], want[~missing])
    assert (got[:, count - 1:] == 7).all()
    assert not missing.any() or found == 4
    assert missing.any() or not surely
    store.wait_us = 0
    scan(store, q, metric, after[:, :count - 1])
    assert status() == 0 and torch.equal(after, want)


def test_a_wait_is_not_negative():
    from vectorlink_gpu import QuantizedVectors, _lib
    store = QuantizedVectors.from_vectors(torch.ones((3, 8), device=DEV))
    store.wait_us = -1
    with pytest.raises(_lib.VlError):
        store.distances(torch.ones((1, 8), device=DEV))
