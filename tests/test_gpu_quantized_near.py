"""Rows held in 8 bits: distances of near and of equal rows, against whole-number arithmetic without any rounding."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = 149          # every fp32 number is a whole multiple of 2^-149


def whole(x):
    """fp32 numbers as whole numbers of 2^-149."""
    return [int(v * 2.0 ** 75) << 74 if v >= 2.0 ** -50 else int(v * 2.0 ** UNIT) for v in np.asarray(x, dtype=np.float64).ravel()]


def held(store):
    return store.codes.cpu().numpy().astype(np.int64)[:, :store.dim], whole(store.scales.cpu().numpy())


def check_l2(got, queries, rows):
    """Every distance in `got` [queries, rows] against the exact one of the held rows.

    With h = 2^-24: results of at least 2^-16 of a + b = |q|^2 + |r|^2 are made in fp32.  The first number of a + b less
    that of 2 t is rounded (h of it), and so is the result (h of it).  What is behind both, parts of numbers cut to 20 bits, is
    below 9/8 2^-19 (a + b), so the first is at most 1 + 9/8 2^-3 < 1.15 of the result.  The parts are rounded when they are made
    and in each of their three sums, h 2^-19 (a + b) or 9/8 of that each time, 4.3 2^-3 < 0.55 of h of the result.  Together
    less than 2 3/4 h.  Smaller results are made in 64 bits of three terms, each of which and whose sums are off by 2^-53
    of the terms, four times at most, then rounded (h).  Both are covered by the sum of the bounds.  What is past the
    largest number of 32 bits is an infinity."""
    (qc, qs), (rc, rs) = queries, rows
    dots, qn, rn = qc @ rc.T, (qc * qc).sum(1), (rc * rc).sum(1)
    got = got.cpu().numpy()
    assert not np.isnan(got).any()
    worst, past = 0.0, (2 ** 25 - 1) << (103 + 2 * UNIT)          # half a step past the largest number
    for i in range(len(qs)):
        g = whole(np.where(np.isinf(got[i]), 0.0, got[i]))
        for j in range(len(rs)):
            (dot, a, b) = int(dots[i, j]), int(qn[i]), int(rn[j])
            terms = (qs[i] - rs[j]) ** 2 * dot, qs[i] ** 2 * (a - dot), rs[j] ** 2 * (b - dot)
            want = sum(terms)
            assert want == qs[i] ** 2 * a + rs[j] ** 2 * b - 2 * qs[i] * rs[j] * dot and want >= 0
            if want == 0:
                assert g[j] == 0, (i, j, got[i, j])
                continue
            # the bounds are taken times 2^51, to stay with whole numbers; half a step of the smallest fp32 number in the end
            slack = (want << 27) * 7 // 4 + 2 * sum(map(abs, terms))
            if np.isinf(got[i, j]) or (want << 51) - slack > past << 51:
                assert np.isinf(got[i, j]) and got[i, j] > 0 and (want << 51) + slack >= past << 51, (i, j, got[i, j])
                continue
            off = abs((g[j] << UNIT) - want)
            bound = (want << 27) + slack + (1 << (UNIT + 50))
            assert off << 51 <= bound, (i, j, got[i, j], float(want) / 2.0 ** (2 * UNIT), off / want)
            worst = max(worst, off / want)
    return worst


def base(count, dim, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((count, dim), generator=g) * scale


def relatives(x, seed):
    """Rows near those of x: longer and shorter copies, copies with noise, both, and rows of the opposite direction."""
    out = [x, -x, 3.0 * x, -0.25 * x]
    for k, e in enumerate((3e-1, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-7)):
        noise = base(*x.shape, seed + k) * x.abs().mean()
        out += [x * (1 + e), x * (1 - e), x + e * noise, (1 + e) * x + e * e * noise]
    return torch.cat(out)


@pytest.mark.parametrize("dim", [1, 7, 50, 96, 768, 1024, 1040, 1536])
@pytest.mark.parametrize("scale", [1.0, 255.0, 1e-15, 1e15, 1e25])
def test_near_rows(dim, scale):
    from vectorlink_gpu import QuantizedVectors
    x = base(6, dim, dim, scale)
    store = QuantizedVectors.from_vectors(relatives(x, dim + 1).to(DEV))
    q = QuantizedVectors.from_vectors(x.to(DEV))
    got = store.distances(q, metric="l2")
    check_l2(got, held(q), held(store))
    ids = torch.arange(len(store), dtype=torch.int32, device=DEV).repeat(6, 1)
    assert torch.equal(store.calculate_distances(q, ids, metric="l2"), got)
    # either side first
    assert torch.equal(q.distances(store, metric="l2").t(), got)


@pytest.mark.parametrize("dim", [2, 50, 96, 384, 768, 1024, 1536])
def test_equal_rows_are_at_distance_zero(dim):
    """A row to itself, and to the same row elsewhere, whatever kernel makes the distance and wherever it comes to lie."""
    from vectorlink_gpu import QuantizedVectors
    x = torch.cat([base(700, dim, dim), base(300, dim, dim + 1).mul_(100.0).round_()]).to(DEV)
    store = QuantizedVectors.from_vectors(torch.cat([x, x]))
    itself = torch.arange(1000, device=DEV)
    for q in (x, x[:16], x[:200].contiguous(), QuantizedVectors.from_vectors(x)):
        count = len(q)
        d = store.distances(q, metric="l2")
        assert not d[itself[:count], itself[:count]].any() and not d[itself[:count], itself[:count] + 1000].any()
        assert (d > 0).sum() >= count * 2000 - 2 * count - 100          # (short rows of few values may meet)
        ids = torch.stack([itself[:count], itself[:count] + 1000], 1).to(torch.int32)
        assert not store.calculate_distances(q, ids, metric="l2").any()


def test_near_rows_are_put_in_order():
    """Copies that grow away from a row step by step: the distances rise with them, as those of the held rows do."""
    from vectorlink_gpu import QuantizedVectors
    x = base(1, 128, 3)
    grown = torch.cat([x * (1 + 2.0 ** -20 * k) for k in range(200)])
    store = QuantizedVectors.from_vectors(grown.to(DEV))
    d = store.distances(x.to(DEV), metric="l2")[0].double()
    s = store.scales.double()
    same = (store.codes == store.codes[0]).all(1)
    assert same.sum() > 100
    want = (s - s[0]) ** 2 * int(store.norms[0])
    assert ((d - want).abs() <= want * 2.0 ** -24 * 1.125)[same].all()


@pytest.mark.parametrize("dim", [1, 7, 96, 768, 1536])
@pytest.mark.parametrize("scale", [1.0, 1e-15, 1e15])
def test_products_are_rounded_once(dim, scale):
    """The product of the scales has 48 digits, the whole number up to 24: all of them count.  With h = 2^-24, the part behind
    24 digits of the scales' product is rounded by h^2 of the result, the result by h of itself."""
    from vectorlink_gpu import QuantizedVectors
    (q, store) = (QuantizedVectors.from_vectors(base(n, dim, n + dim, scale).to(DEV)) for n in (40, 300))
    (qc, qs), (rc, rs) = held(q), held(store)
    dots, got = qc @ rc.T, store.product(q).cpu().numpy()
    assert np.array_equal(q.product(store).t().cpu().numpy(), got)
    for i in range(40):
        for j in range(300):
            want = qs[i] * rs[j] * int(dots[i, j])
            off = abs((whole([abs(got[i, j])])[0] << UNIT) - abs(want))
            assert (got[i, j] < 0) == (want < 0) or want == 0
            assert off << 48 <= (abs(want) << 24) + abs(want) + (1 << (UNIT + 47)), (i, j, got[i, j])
