"""Rows held in 8 bits: calls large enough that every CTA and warp has several pieces of work, against the plain form.

The plain form is made on the device in 64 bits: whole-number products are exact there."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MAXINT = 2147483647
MAXFLOAT = 3.4028e37
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134 + 2.0 ** -149, torch.float16: 2.0 ** -25 + 2.0 ** -149}


def rows(count, dim, seed, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn((count, dim), generator=g, device=DEV).to(dtype)


def quantise(x):
    """codes and scales of `x` in 64 bits, codes [n, dim]."""
    x = x.double()
    bad = ~x.isfinite().all(1)
    x = torch.where(bad.unsqueeze(1), 0.0, x)
    scales = (x.abs().amax(1) / 127.0).float()
    s = scales.double().unsqueeze(1)
    codes = torch.where(s > 0, (x / s).round(), 0.0).clamp(-127, 127)
    return codes, torch.where(bad, float("nan"), scales).float()


def held(store):
    return store.codes[:, :store.dim].double(), store.scales.double()


def check_scores(got, queries, stored, metric):
    """With h = 2^-24.  Products: h of the result (and half a step of 16 bits, of a value with two such roundings).  Cosine: 1/2 - sh f is
    rounded (h of a number that the rest, below 2^-23 |t|, takes to the result), the rest (2^-48 |t|), the result (h): 2 h of
    it and 2^-44 (1 + |t|).  l2: 2 3/4 h of the result, or one rounding where it is below 2^-16 (a + b), of three terms in 64
    bits; the plain form below makes it of the same terms, so both together are off by 2^-48 of their magnitudes at most.
    Below the smallest normal number h of a number is less than its rounding, half of the smallest step: 2^-150 in fp32, 2^-134 in
    bf16 and 2^-25 in fp16, whose rounding follows that of fp32 (here the products of two rows of 1e-30 come to 1e-60)."""
    (qc, qs), (rc, rs) = queries, stored
    h = 2.0 ** -24
    qn, rn = (qc * qc).sum(1, keepdim=True), (rc * rc).sum(1)
    step = max(1, 30_000_000 // max(1, rc.shape[0]))
    for lo in range(0, qc.shape[0], step):
        c, s, n = qc[lo:lo + step], qs[lo:lo + step].unsqueeze(1), qn[lo:lo + step]
        dots = c @ rc.T
        t = s * rs * dots
        if metric == "product":
            half = HALF_STEP[got.dtype]
            want, bound = t, t.abs() * (h * (1 + 2.0 ** -20) if got.dtype == torch.float32 else (half + 2 * h) * 1.01)
        elif metric == "cosine":
            want = ((1.0 - t) * 0.5).clamp(0.0, 1.0)
            bound = 2 * h * want + 2.0 ** -44 * (1 + t.abs())
        else:
            terms = (s - rs) ** 2 * dots, s * s * (n - dots), rs * rs * (rn - dots)
            want = (terms[0] + terms[1] + terms[2]).clamp_min(0.0)
            bound = 2.75 * h * want + 2.0 ** -48 * (terms[0].abs() + terms[1].abs() + terms[2].abs())
        mine, bound = got[lo:lo + step].double(), bound + SMALLEST[got.dtype]
        nan = want.isnan()
        assert torch.equal(mine.isnan(), nan)
        ok = nan | ((mine - want).abs() <= bound)
        assert ok.all(), (metric, lo, int((~ok).sum()), (~ok).nonzero()[0].tolist(), mine[~ok][0].item(), want[~ok][0].item())


# What is to be met (with 148 SMs): queries that stay in shared memory in blocks of 16, 48 and 128, and ones that stream in blocks of
# 112 (four accumulators, a finishing group for a tile), 144 and 160 (three, two groups for a tile), 176 to 256 (two); 4 to 28 tiles for a
# CTA; and several blocks of queries for a CTA, of both kinds.
SHAPES = [(16, 60_007, 96), (48, 60_007, 96), (1000, 60_007, 32), (1000, 30_007, 300), (100, 60_007, 1536), (150, 100_003, 640), (320, 40_001, 640),
          (170, 60_001, 640), (700, 60_007, 520), (2500, 20_011, 520), (20_000, 300, 16), (40_000, 700, 16), (40_000, 300, 528)]


@pytest.mark.parametrize("nq,count,dim", SHAPES)
@pytest.mark.parametrize("metric", ["product", "cosine", "l2"])
@pytest.mark.parametrize("ragged", [False, True])
def test_scores_of_many_tiles(nq, count, dim, metric, ragged):
    """Rows of ordinary length with some among them that are zero, far longer, near a query or its copy, too small for fp32, or no
    numbers; the same in the queries.  Results on sectors, and off them."""
    from vectorlink_gpu import QuantizedVectors
    x, q = rows(count, dim, 1), rows(nq, dim, 2)
    if metric == "cosine":
        x, q = torch.nn.functional.normalize(x, dim=1), torch.nn.functional.normalize(q, dim=1)
    x[5::997] = 0.0
    x[6::1013] *= 300.0
    x[7::1009] = q[0] * (1 + 1e-4)
    x[8::1019] = q[nq // 2]
    x[count // 2] *= 1e-30
    x[count - 1, 0] = float("nan")
    if nq > 200:
        q[3] *= 1e-30
        q[7] = 0.0
        q[nq - 1, dim - 1] = float("inf")
    store, asked = QuantizedVectors.from_vectors(x), QuantizedVectors.from_vectors(q)
    for dtype in ((torch.float32, torch.bfloat16, torch.float16) if metric == "product" else (torch.float32,)):
        stride = count + 1 if ragged else (count + 15) // 16 * 16
        out = torch.full((nq, stride), 7.0, dtype=dtype, device=DEV)
        place = out[:, stride - count:] if ragged else out[:, :count]
        if metric == "product":
            store.product(q, out=place)
        else:
            store.distances(q, metric=metric, out=place)
        assert (out[:, :stride - count] == 7).all() if ragged else (out[:, count:] == 7).all()
        check_scores(place, held(asked), held(store), metric)


def test_more_results_than_32_bits_count():
    from vectorlink_gpu import QuantizedVectors
    (nq, count, dim) = (33_000, 66_001, 48)
    store, q = QuantizedVectors.from_vectors(rows(count, dim, 1)), QuantizedVectors.from_vectors(rows(nq, dim, 2))
    got = store.product(q, dtype=torch.bfloat16)
    assert got.numel() > 2 ** 31
    for lo in (0, 16_000, nq - 64):
        part = QuantizedVectors(64, dim, device=DEV)
        part.codes.copy_(q.codes[lo:lo + 64])
        part.scales.copy_(q.scales[lo:lo + 64])
        part.norms.copy_(q.norms[lo:lo + 64])
        check_scores(got[lo:lo + 64], held(part), held(store), "product")


@pytest.mark.parametrize("count,dim,dtype", [(200_003, 8, torch.float32), (200_003, 100, torch.bfloat16), (160_003, 200, torch.float16), (90_001, 200, torch.float32),
                                             (80_003, 700, torch.bfloat16), (40_003, 700, torch.float32), (40_003, 800, torch.float16)])
def test_more_rows_than_warps(count, dim, dtype):
    """Written as a block and to places (some named again, some none), read as a range and at ids."""
    from vectorlink_gpu import QuantizedVectors, _lib
    x = rows(count, dim, dim, dtype)
    x[11::5003] = 0.0
    x[12::5003, dim - 1] = float("inf")
    x[13::5003] *= 1e-7 if dtype == torch.float16 else 1e-38
    (codes, scales) = quantise(x)
    values = codes * scales.double().unsqueeze(1)
    _lib.read_status(DEV)

    def same(store, places, c, s):
        assert torch.equal(store.codes[places, :dim].double(), c) and not store.codes[:, dim:].any()
        assert torch.equal(store.scales[places].nan_to_num(-1.0), s.nan_to_num(-1.0))
        assert torch.equal(store.norms[places].double(), (c * c).sum(1))

    def read_as(got, want):
        half = HALF_STEP[got.dtype]
        bound = want.abs() * (half + (2.0 ** -24 if half > 2.0 ** -24 else 0.0)) * (1 + 2.0 ** -20) + SMALLEST[got.dtype]
        assert torch.equal(got.isnan(), want.isnan()) and ((got.double() - want).abs() <= bound)[~want.isnan()].all()

    store = QuantizedVectors.from_vectors(x)
    same(store, slice(None), codes, scales)
    for out_type in HALF_STEP:
        read_as(store.read(dtype=out_type), values)
    read_as(store.read(rows=(3, count - 2)), values[3:count - 2])
    g = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.randint(0, count, (count,), generator=g, device=DEV).to(torch.int32)
    ids[::17] = MAXINT
    other = QuantizedVectors(count, dim, device=DEV)
    other.write(x, ids=ids)
    order = torch.arange(count, device=DEV)
    last = torch.full((count + 1,), -1, dtype=torch.int64, device=DEV)
    last.scatter_reduce_(0, torch.where(ids == MAXINT, count, ids).long(), order, "amax")
    last = last[:count]
    places = (last >= 0).nonzero()[:, 0]
    same(other, places, codes[last[places]], scales[last[places]])
    untouched = (last < 0).nonzero()[:, 0]
    assert not other.codes[untouched].any() and not other.scales[untouched].any() and (other._owner == -1).all()
    got = store.read(ids=ids, dtype=torch.bfloat16)
    assert not got[::17].any()
    kept = (ids != MAXINT).nonzero()[:, 0]
    read_as(got[kept], values[ids[kept].long()])
    assert _lib.read_status(DEV) == 0


@pytest.mark.parametrize("lists,width,dim", [(40_001, 5, 8), (40_001, 33, 100), (40_001, 3, 300), (40_001, 40, 40), (40_001, 2, 700), (38_000, 2, 1500), (40_001, 2, 1600)])
@pytest.mark.parametrize("metric", ["cosine", "l2"])
def test_more_lists_than_warps(lists, width, dim, metric):
    """Every list against the scan of the rows that it names, whose results are checked above: the same bits."""
    from vectorlink_gpu import QuantizedVectors, _lib
    count = 500
    x, q = rows(count, dim, 1), rows(lists, dim, 2, torch.bfloat16)
    if metric == "cosine":
        x, q = torch.nn.functional.normalize(x, dim=1), torch.nn.functional.normalize(q.float(), dim=1).bfloat16()
    x[5] = 0.0
    x[6, 1] = float("nan")
    q[9] = 0.0
    store = QuantizedVectors.from_vectors(x)
    g = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(0, count, (lists, width), generator=g, device=DEV).to(torch.int32)
    none = torch.rand((lists, width), generator=g, device=DEV) < 0.1
    ids[none] = MAXINT
    ids[4] = MAXINT
    none[4] = True
    _lib.read_status(DEV)
    got = store.calculate_distances(q, ids, metric=metric)
    scan = store.distances(q, metric=metric)
    check_scores(scan, held(QuantizedVectors.from_vectors(q)), held(store), metric)
    want = torch.where(none, MAXFLOAT, torch.gather(scan, 1, torch.where(none, 0, ids).long()))
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(-1.0), want.nan_to_num(-1.0))
    assert _lib.read_status(DEV) == 0
