"""Lists of ids longer than a 32-bit length (no GPU calls)."""
import ctypes

import pytest
import torch


def test_lists_of_more_than_a_length_can_say(built_lib, monkeypatch):
    """A length that does not fit is refused; it is not cut to 32 bits.  The ids take no memory: one element, seen many times."""
    from vectorlink_gpu import QuantizedVectors, quantized
    store = QuantizedVectors(10, 24, device="cpu")
    monkeypatch.setattr(quantized._lib, "require_cuda", lambda *t: None)

    def reached():
        raise RuntimeError("reached the library")
    monkeypatch.setattr(quantized, "lib", reached)
    # no list is copied or allocated before its length is looked at
    monkeypatch.setattr(torch.Tensor, "contiguous", lambda t: t)
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda t, shape, **kw: torch.empty(1).expand(shape))
    for width in (2 ** 30 + 1, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5):
        ids = torch.zeros((1, 1), dtype=torch.int32).expand(1, width)
        with pytest.raises(AssertionError, match="list"):
            store.calculate_distances(torch.zeros(1, 24), ids)


def test_the_library_refuses_long_lists(built_lib):
    from vectorlink_gpu import _lib
    p = ctypes.c_void_p(256)
    for width in (2 ** 30 + 1, 2 ** 31 - 1, -1):
        rc = _lib.lib().vl_quant_listed(p, 0, 24, p, p, p, 1, p, p, p, 10, 24, 32, p, width, p, 0, p, None)
        assert rc == -1 and b"size" in _lib.lib().vl_last_error()
