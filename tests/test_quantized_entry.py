"""Rows held in 8 bits: what the C entry points refuse before anything is launched (no GPU calls)."""
import ctypes

import pytest

WRITE = dict(rows=256, type=0, m=4, dim=24, ld=24, ids=None, first_row=0, codes=256, scales=256, norms=256, n=10, code_ld=32, owner=256,
             status=256, stream=None)
READ = dict(codes=256, scales=256, n=10, dim=24, code_ld=32, ids=None, first_row=0, m=4, out=256, type=0, out_ld=24, status=256, stream=None)
SCORES = dict(queries=256, q_type=0, q_ld=24, q_codes=256, q_scales=256, q_norms=256, nq=4, codes=256, scales=256, norms=256, n=10, dim=24,
              code_ld=32, row_lo=0, row_hi=10, out=256, type=0, out_ld=10, metric=0, status=256, stream=None)
LISTED = dict(queries=256, q_type=0, q_ld=24, q_codes=256, q_scales=256, q_norms=256, nq=4, codes=256, scales=256, norms=256, n=10, dim=24,
              code_ld=32, ids=256, w=3, out=256, metric=0, status=256, stream=None)


def refusal(name, arguments, **changed):
    """What the library says to a call whose pointers are numbers: it has to refuse on the host, before it reads any."""
    from vectorlink_gpu import _lib
    assert set(changed) <= set(arguments)
    rc = getattr(_lib.lib(), name)(*{**arguments, **changed}.values())
    assert rc == -1, (name, changed, rc, _lib.lib().vl_last_error())
    return _lib.lib().vl_last_error().decode()


@pytest.mark.parametrize("name,arguments,changed", [
    ("vl_quant_write", WRITE, dict(rows=258)),
    ("vl_quant_write", WRITE, dict(rows=257, type=1)),
    ("vl_quant_write", WRITE, dict(rows=257, type=2)),
    ("vl_quant_write", WRITE, dict(scales=258)),
    ("vl_quant_write", WRITE, dict(norms=257)),
    ("vl_quant_write", WRITE, dict(status=258)),
    ("vl_quant_write", WRITE, dict(ids=258)),
    ("vl_quant_write", WRITE, dict(ids=256, owner=257)),
    ("vl_quant_read", READ, dict(out=258)),
    ("vl_quant_read", READ, dict(out=257, type=1)),
    ("vl_quant_read", READ, dict(out=257, type=2)),
    ("vl_quant_read", READ, dict(scales=258)),
    ("vl_quant_read", READ, dict(status=257)),
    ("vl_quant_read", READ, dict(ids=258)),
    ("vl_quant_scores", SCORES, dict(queries=258)),
    ("vl_quant_scores", SCORES, dict(queries=257, q_type=1)),
    ("vl_quant_scores", SCORES, dict(queries=257, q_type=2)),
    ("vl_quant_scores", SCORES, dict(queries=None, q_scales=258)),
    ("vl_quant_scores", SCORES, dict(nq=17, q_norms=258)),
    ("vl_quant_scores", SCORES, dict(scales=257)),
    ("vl_quant_scores", SCORES, dict(norms=258)),
    ("vl_quant_scores", SCORES, dict(status=258)),
    ("vl_quant_listed", LISTED, dict(queries=258)),
    ("vl_quant_listed", LISTED, dict(queries=257, q_type=1)),
    ("vl_quant_listed", LISTED, dict(queries=None, q_scales=258)),
    ("vl_quant_listed", LISTED, dict(queries=None, q_norms=257)),
    ("vl_quant_listed", LISTED, dict(scales=258)),
    ("vl_quant_listed", LISTED, dict(norms=258)),
    ("vl_quant_listed", LISTED, dict(ids=258)),
    ("vl_quant_listed", LISTED, dict(out=258)),
    ("vl_quant_listed", LISTED, dict(status=257)),
])
def test_places_that_are_not_aligned_to_their_elements(built_lib, name, arguments, changed):
    message = refusal(name, arguments, **changed)
    assert name in message and "aligned" in message


def test_rows_of_a_result_that_overlap(built_lib):
    for out_ld in (23, 0, -24):
        assert "overlap" in refusal("vl_quant_read", READ, out_ld=out_ld)
    for out_ld in (9, 0, -10):
        assert "overlap" in refusal("vl_quant_scores", SCORES, out_ld=out_ld)


def test_waits_that_are_none_or_too_long(built_lib):
    wait = {**{k: v for k, v in SCORES.items() if k not in ("status", "stream")}, "wait_us": 0, "status": 256, "stream": None}
    for wait_us in (-1, 2_000_001, 2 ** 31 - 1):
        assert "wait" in refusal("vl_quant_scores_wait", wait, wait_us=wait_us)
    assert "aligned" in refusal("vl_quant_scores_wait", wait, out=258)
