"""Vectors held in 8 bits: a quarter of the memory, and a quarter of the bytes that a scan has to read.

The reference keeps fp32 rows only.  A `QuantizedVectors` holds a row as whole numbers in [-127, 127] and one fp32 scale
(max|x| / 127), takes rows as they come (written as a block or to listed places), gives them back, and scores queries
against all rows of a range or against listed ids.  Queries are held in 8 bits as well, one scale each, and the
products of the whole numbers are summed exactly, so a pair has the same bits in `distances` and in
`calculate_distances`, and rows that are held alike are at a squared distance of exactly 0.  The distances are those of
the rows as they are held: approximations (0.4 % of the largest element, per element) of the fp32 rows' distances, to be
scored again with `kernels.calculate_distances` where that matters.

A row that holds an infinity or a NaN is held as NaN: so is everything that is made of it.  Ids outside the store, and a
wait inside a scan that ran out, are reported in the device's status word (`_lib.read_status`), like those of the other
kernels; results that were not made because of such a wait are NaN.  A store belongs to the device that it was made on; its
calls run on torch's current stream there.  A result that the caller provides must not lie in memory that the call
reads.  No gradient passes through any of this: results are data.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from ._lib import check, lib
from .constants import MAXINT
from .kernels import metric_code

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
PRODUCT = 2            # VL_QUANT_PRODUCT: the metric code of a plain product
MAX_DIM = 131072       # 127^2 * dim has to fit 32 bits
MAX_LIST = 1 << 30     # ids of one list
LISTED_ROUNDS = 1536   # columns up to which the scoring of listed ids rounds its queries in registers
FEW_QUERIES = (16, 4096)   # queries, and columns of them, up to which a scan rounds its queries itself
FEW_ROWS = 64          # rows up to which a write to places is one launch


class QuantizedVectors:
    """`codes` int8 [count, dim to the next multiple of 16] (zeros behind `dim`), `scales` fp32 [count] and `norms` int32
    [count] (sum of squared codes).  Rows that were never written are zero."""

    wait_us = 0     # longest wait inside a scan, in microseconds, up to two seconds (0)

    def __init__(self, count: int, dim: int, device="cuda"):
        self._allocate(count, dim, device, torch.zeros)

    def _allocate(self, count: int, dim: int, device, make) -> None:
        assert 0 <= count < MAXINT and 1 <= dim <= MAX_DIM
        self.dim = dim
        self.count = count
        self._columns = (dim + 15) // 16 * 16
        self.codes = make((count, self._columns), dtype=torch.int8, device=device)
        self.scales = make((count,), dtype=torch.float32, device=device)
        self.norms = make((count,), dtype=torch.int32, device=device)
        # during a write: the last row that names a place
        self._owner = torch.full((count,), -1, dtype=torch.int32, device=device)
        self.device = self.codes.device
        # (made here, so that it exists before a call is captured)
        self._status = _lib.status_word(self.device) if self.codes.is_cuda else None

    @classmethod
    def from_vectors(cls, vectors: Tensor) -> "QuantizedVectors":
        """All rows of `vectors` [count, dim], fp32, bf16 or fp16."""
        _lib.require_cuda(vectors)
        assert vectors.dim() == 2, f"rows: [count, dim] expected, got {tuple(vectors.shape)}"
        store = cls.__new__(cls)
        store._allocate(vectors.size(0), vectors.size(1), vectors.device, torch.empty)      # the write fills all of it
        store.write(vectors)
        return store

    def __len__(self) -> int:
        return self.count

    # Argument checks.  A call's own work is a few microseconds on the device, so these are kept few and cheap.

    def _here(self, t: Tensor) -> None:
        if t.device != self.device:
            _lib.require_cuda(t)
            raise AssertionError(f"rows are held on {self.device}, got a tensor on {t.device}")

    def _rows(self, t: Tensor, what: str) -> Tensor:
        """`t` as rows of `dim` elements that lie next to one another (a column slice stays where it is)."""
        shape = t.shape
        assert len(shape) == 2 and shape[1] == self.dim, f"{what}: [rows, {self.dim}] expected, got {tuple(shape)}"
        assert t.dtype in TYPES, f"{what}: fp32, bf16 or fp16 expected, got {t.dtype}"
        self._here(t)
        return t if shape[1] == 1 or t.stride(1) == 1 else t.contiguous()

    def _range(self, rows: Optional[Tuple[int, int]]) -> Tuple[int, int]:
        if rows is None:
            return 0, self.count
        (lo, hi) = rows
        assert 0 <= lo <= hi <= self.count, f"rows {lo}..{hi} outside 0..{self.count}"
        return lo, hi

    def _ids(self, ids: Tensor, dims: int) -> Tensor:
        assert ids.dtype == torch.int32 and ids.dim() == dims
        self._here(ids)
        return ids.contiguous()

    def _result(self, out: Optional[Tensor], rows: int, cols: int, dtype) -> Tensor:
        if out is None:
            assert dtype in TYPES, f"fp32, bf16 or fp16 expected, got {dtype}"
            return self.codes.new_empty((rows, cols), dtype=dtype)
        assert out.dtype in TYPES and tuple(out.shape) == (rows, cols), f"result of {(rows, cols)} expected, got {tuple(out.shape)}"
        assert (cols <= 1 or out.stride(1) == 1) and (rows <= 1 or out.stride(0) >= cols), "rows of the result have to lie apart, their elements together"
        self._here(out)
        return out

    def _queries(self, queries: Union[Tensor, "QuantizedVectors"], rounded: int):
        """How many, the library's arguments (rows to quantise or none, their type and stride, and where the codes, scales
        and sums of squares are or go), and what has to live until the call.  Up to `rounded` queries need no such place."""
        if isinstance(queries, QuantizedVectors):
            assert queries.dim == self.dim
            self._here(queries.codes)
            return queries.count, (None, 0, 0, queries.codes.data_ptr(), queries.scales.data_ptr(), queries.norms.data_ptr()), queries
        x = self._rows(queries, "queries")
        (rows, ld) = (x.size(0), x.stride(0))
        if rows <= rounded:
            return rows, (x.data_ptr(), TYPES[x.dtype], ld, None, None, None), x
        codes, scales = rows * self._columns, (4 * rows + 15) // 16 * 16
        buffer = self.codes.new_empty(codes + 2 * scales)
        at = buffer.data_ptr()
        return rows, (x.data_ptr(), TYPES[x.dtype], ld, at, at + codes, at + codes + scales), (x, buffer)

    def _held(self):
        """The library's arguments that say what is held."""
        return self.codes.data_ptr(), self.scales.data_ptr(), self.norms.data_ptr(), self.count, self.dim, self._columns

    def _run(self, name: str, *args) -> None:
        """One call of the library with the status word and torch's current stream of the rows' device, which is made the
        current one for it."""
        _lib.require_cuda(self.codes)
        index = self.device.index
        status, stream = self._status.data_ptr(), torch._C._cuda_getCurrentRawStream(index)
        call = getattr(lib(), name)
        if torch.cuda.current_device() == index:
            check(call(*args, status, stream), name)
        else:
            with torch.cuda.device(index):
                check(call(*args, status, stream), name)

    def write(self, vectors: Tensor, ids: Optional[Tensor] = None, first_row: int = 0) -> None:
        """Row r of `vectors` (fp32, bf16 or fp16; a column slice of a wider matrix is read where it lies) goes to
        place ids[r] (int32), or to first_row + r.  A row with the id MAXINT is skipped; of rows with the same id the
        last one is kept; an id outside the store is skipped and reported in the status word.  Writes to one place from
        several streams at once are the caller's to order, like any use of a tensor."""
        x = self._rows(vectors, "write")
        m = x.size(0)
        places = None
        if ids is not None:
            assert first_row == 0, "rows go to their ids or to a block, not both"
            ids = self._ids(ids, 1)
            assert ids.size(0) == m
            places = ids.data_ptr()
        else:
            assert 0 <= first_row and first_row + m <= self.count, f"rows {first_row}..{first_row + m} outside 0..{self.count}"
        if m == 0:
            return
        self._run("vl_quant_write", x.data_ptr(), TYPES[x.dtype], m, self.dim, x.stride(0), places, first_row, self.codes.data_ptr(),
                  self.scales.data_ptr(), self.norms.data_ptr(), self.count, self._columns, self._owner.data_ptr())
        if places is not None and m > FEW_ROWS:
            _lib.LAUNCHES += 1      # which row keeps a place

    def read(self, ids: Optional[Tensor] = None, rows: Optional[Tuple[int, int]] = None, dtype=torch.float32,
             out: Optional[Tensor] = None) -> Tensor:
        """The held values of the rows `ids` (int32; zeros where MAXINT), of the rows [lo, hi), or of all."""
        assert ids is None or rows is None, "rows are read by their ids or as a range, not both"
        places = None
        if ids is not None:
            ids = self._ids(ids, 1)
            places = ids.data_ptr()
            (lo, count) = (0, ids.size(0))
        else:
            (lo, hi) = self._range(rows)
            count = hi - lo
        out = self._result(out, count, self.dim, dtype)
        if count:
            self._run("vl_quant_read", self.codes.data_ptr(), self.scales.data_ptr(), self.count, self.dim, self._columns, places, lo, count,
                      out.data_ptr(), TYPES[out.dtype], out.stride(0))
        return out

    def _scores(self, queries, rows, metric: int, dtype, out: Optional[Tensor]) -> Tensor:
        (lo, hi) = self._range(rows)
        (few, columns) = FEW_QUERIES
        (count, q, _alive) = self._queries(queries, few if self._columns <= columns else 0)
        out = self._result(out, count, hi - lo, dtype)
        if count and hi > lo:
            self._run("vl_quant_scores_wait", *q, count, *self._held(), lo, hi, out.data_ptr(), TYPES[out.dtype], out.stride(0), metric,
                      self.wait_us)
            if q[0] is not None and q[3] is not None:
                _lib.LAUNCHES += 1      # the queries' codes
        return out

    def product(self, queries: Union[Tensor, "QuantizedVectors"], rows: Optional[Tuple[int, int]] = None, dtype=torch.float32,
                out: Optional[Tensor] = None) -> Tensor:
        """[queries, hi - lo]: the inner product of every query with every row of [lo, hi), both as held in 8 bits.
        `out` (its type is the result's) may be a slice of a wider matrix, so that a scan can go range by range."""
        return self._scores(queries, rows, PRODUCT, dtype, out)

    def distances(self, queries: Union[Tensor, "QuantizedVectors"], rows: Optional[Tuple[int, int]] = None, metric="cosine",
                  out: Optional[Tensor] = None) -> Tensor:
        """fp32 [queries, hi - lo]: the distance (cosine of unit vectors, or squared l2) of every query to every row of
        [lo, hi)."""
        assert out is None or out.dtype == torch.float32
        return self._scores(queries, rows, metric_code(metric), torch.float32, out)

    def calculate_distances(self, queries: Union[Tensor, "QuantizedVectors"], beams: Tensor, distances_out: Optional[Tensor] = None,
                            metric="cosine") -> Tensor:
        """`kernels.calculate_distances` over the held rows: out[i, j] = distance(queries[i], row beams[i, j]), MAXFLOAT
        where beams[i, j] == MAXINT."""
        (count, q, _alive) = self._queries(queries, MAXINT if self._columns <= LISTED_ROUNDS else 0)
        beams = self._ids(beams, 2)
        (rows, width) = beams.shape
        assert rows == count
        # (the library takes a list's length as an int: a longer one would arrive cut to 32 bits)
        assert width <= MAX_LIST, f"list of up to {MAX_LIST} ids expected, got {width}"
        out = distances_out
        if out is None:
            out = self.codes.new_empty((rows, width), dtype=torch.float32)
        else:
            assert out.is_contiguous() and out.dtype == torch.float32 and out.shape == beams.shape
            self._here(out)
        if rows and width:
            self._run("vl_quant_listed", *q, count, *self._held(), beams.data_ptr(), width, out.data_ptr(), metric_code(metric))
            if q[0] is not None and q[3] is not None:
                _lib.LAUNCHES += 1      # the queries' codes
        return out
