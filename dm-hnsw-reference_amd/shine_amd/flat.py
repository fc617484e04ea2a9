"""Flat scoring: every record of a table against every query, on torch tensors (C ABI: shine_flat_*).

The complement of the graph search for filters that leave it too few records, tables too small for a graph and candidate
lists.  Records and queries are held as 8-bit codes with a scale each: answers are exact for the codes, not for the rows
(of the ten best of 200,000 normal rows of 96 to 768 components, 97.5 to 98 % are found).

    table = FlatTable(rows, metric="l2")                 # quantised once
    values, ids = search(table, queries, 10, allow=bits) # the k best allowed records of every query

or step by step, with the score matrix in hand:

    s = scores(table, queries)
    s = adjust(s, bias=boost, allow=bits, seen=shown, repetition=r, frequency=f, presence=p)
    values, ids = topk(s, 10)

Tensors are CUDA tensors of torch.float32, float16 or bfloat16 with unit stride along their last dimension; calls run on
the current stream of the tensors' device and do not wait for it.  There are no gradients: tensors that require one are
refused unless under torch.no_grad().
"""
from __future__ import annotations

import ctypes as C

from . import _lib as L

MAX_K = 256
MAX_DIM = 16384
MAX_ROWS = 2 ** 32 - 1  # of queries or scores in a call: the C entries count them in 32 bits

_torch = _current = None
_elems = {}


def _t():
    global _torch, _current
    if _torch is None:
        import torch
        # the stream's handle alone where torch gives it: a Stream object costs 2 us a call
        _current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda index: torch.cuda.current_stream(index).cuda_stream)
        _elems.update({torch.float32: L.ELEM_F32, torch.float16: L.ELEM_F16, torch.bfloat16: L.ELEM_BF16})
        _torch = torch  # last: other threads take it as a sign that the rest is there
    return _torch


def _learned(name: str):
    if _torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: flat scoring has none")


def _rows(x, name: str, device=None):
    """(pointer, element type, row stride, rows, width) of a 2-D tensor of rows, or ValueError."""
    torch = _t()
    if not isinstance(x, torch.Tensor) or len(shape := x.shape) != 2:
        raise ValueError(f"{name} must be a 2-D tensor")
    elem = _elems.get(x.dtype)
    if elem is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {x.dtype}")
    index = x.get_device()
    if index < 0 or not x.is_cuda:
        raise ValueError(f"{name} must be on a GPU")
    if device is not None and index != device.index:
        raise ValueError(f"{name} is on {x.device}, not on {device}")
    if x.requires_grad:
        _learned(name)
    n, width = shape
    ld = width
    if not x.is_contiguous():
        ld, unit = x.stride()
        if width > 1 and unit != 1:
            raise ValueError(f"{name} must have unit stride along its last dimension")
        if n < 2:
            ld = width
    return x.data_ptr(), elem, ld, n, width


def _too_many(name: str):
    raise ValueError(f"{name} must have at most {MAX_ROWS} rows")


def _side(x, name: str, dtype, nq: int, width: int | None, device):
    """(pointer, row stride, width) of an adjustment given for each row (nq, width), or shared (1, width) or (width,)."""
    if not isinstance(x, _torch.Tensor) or x.dtype != dtype or x.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    shape = x.shape
    n, w = (1, *shape) if len(shape) == 1 else shape if len(shape) == 2 else (-1, 0)
    if n != 1 and n != nq or n < 0 or (width is not None and w != width):
        raise ValueError(f"{name} must have {'one row or ' + str(nq)} rows" +
                         (f" of {width}" if width is not None else ""))
    ld = w
    if not x.is_contiguous():
        if w > 1 and x.stride(-1) != 1:
            raise ValueError(f"{name} must have unit stride along its last dimension")
        ld = x.stride(0)
    return x.data_ptr(), ld if n > 1 else 0, w


def _adjustment(nq, n, device, bias, allow, seen, repetition, frequency, presence):
    torch = _t()
    a = L.FlatAdjustment()
    if bias is not None:
        a.bias, a.bias_ld, _ = _side(bias, "bias", torch.float32, nq, n, device)
        if bias.requires_grad:
            _learned("bias")
    if allow is not None:
        a.allow, a.allow_ld, _ = _side(allow, "allow", torch.int32, nq, (n + 31) // 32, device)
    if seen is not None:
        a.seen, a.seen_ld, h = _side(seen, "seen", torch.int32, nq, None, device)
        a.seen_n = h if h < 2 ** 32 else 2 ** 32 - 1  # too many are refused by the entry, not taken modulo 2^32 here
    for name, x in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
        if x is not None:
            if seen is None:
                raise ValueError(f"{name} needs seen")
            if not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.device != device or \
                    x.shape != (nq,) or not x.is_contiguous():
                raise ValueError(f"{name} must be a contiguous float32 tensor of {nq} numbers on {device}")
            if x.requires_grad:
                _learned(name)
            setattr(a, name, x.data_ptr())
    return a


def _stream(device) -> int:
    return _current(device.index)


def _workspace(size: int, device):
    return _t().empty(size, dtype=_torch.uint8, device=device) if size else None


def quantize_rows(rows):
    """Rows (n, dim) -> codes int8 (n, dim), a view of rows of code_pitch(dim) bytes, and scales float32 (n,).

    scale = f32(max|x| / 127), code = the integer nearest to x / scale (halves to even): codes * scales[:, None] are the
    rows within half a scale.  A row of zeros has scale 0; a row with an infinity or NaN has scale NaN and codes 0.
    """
    codes, scales, _ = _quantize(rows, False)
    return codes[:, :rows.shape[1]], scales


def code_pitch(dim: int) -> int:
    """Bytes of a row of codes."""
    return (dim + 63) // 64 * 64


def _quantize(rows, norms: bool):
    torch = _t()
    ptr, elem, ld, n, dim = _rows(rows, "rows")
    if not 1 <= dim <= MAX_DIM:
        raise ValueError(f"dim must be in [1, {MAX_DIM}]")
    codes = torch.empty((n, code_pitch(dim)), dtype=torch.int8, device=rows.device)
    scales = torch.empty(n, dtype=torch.float32, device=rows.device)
    half = torch.empty(n, dtype=torch.float32, device=rows.device) if norms else None
    L.check(L.lib().shine_flat_quantize(rows.device.index, ptr, elem, n, dim, ld, codes.data_ptr(), scales.data_ptr(),
                                        half.data_ptr() if norms else None, _stream(rows.device)))
    return codes, scales, half


class FlatTable:
    """Records as 8-bit codes with a scale each, on one GPU.

    metric "ip": a score is the inner product.  metric "l2": the inner product minus half the record's squared norm, so
    that larger is closer; `distances` turns such scores into squared L2 distances.

    codes (n, code_pitch(dim)), scales (n,) and bias ((n,), None for "ip") may be changed in place, not replaced: the calls
    read the memory that the table was made with.
    """

    _PARTS = ("codes", "scales", "bias", "n", "dim", "metric", "device", "_c")

    def __init__(self, rows, metric: str = "ip"):
        if metric not in ("ip", "l2"):
            raise ValueError(f"metric must be 'ip' or 'l2', not {metric!r}")
        self.codes, self.scales, self.bias = _quantize(rows, metric == "l2")
        self.n, self.dim = rows.shape
        self.metric, self.device = metric, rows.device
        self._c = L.FlatTable(self.codes.data_ptr(), self.scales.data_ptr(),
                              self.bias.data_ptr() if metric == "l2" else None, self.n, self.dim, 0)

    def __setattr__(self, name, value):
        if name in self._PARTS and self.__dict__.get(name, value) is not value:  # `table.bias += x` gives the same one back
            raise AttributeError(f"a table's {name} cannot be replaced")
        super().__setattr__(name, value)

    def __delattr__(self, name):
        if name in self._PARTS:
            raise AttributeError(f"a table's {name} cannot be taken away")
        super().__delattr__(name)

    def distances(self, values, queries):
        """Squared L2 distances of the scores `values` (nq, ...) of an "l2" table: max(|q|^2 - 2 value, 0), between the rows
        that the codes of the queries and of the records stand for.  Places without an answer are infinitely far."""
        if self.metric != "l2":
            raise ValueError("the table's scores are inner products")
        queries = queries.to(self.device)
        _queries(self, queries)
        half = _quantize(queries, True)[2].to(values.device)  # -|q|^2 / 2, of the quantised query as in its scores
        values = values.float()
        far = (-2.0 * (half.reshape(-1, *[1] * (values.dim() - 1)) + values)).clamp_min(0.0)
        return far.masked_fill(values == float("-inf"), float("inf"))


def _queries(table, queries):
    if not isinstance(table, FlatTable):
        raise ValueError("table must be a FlatTable")
    ptr, elem, ld, nq, dim = _rows(queries, "queries", table.device)
    if dim != table.dim:
        raise ValueError(f"queries have dim {dim}, the table {table.dim}")
    if nq > MAX_ROWS:
        _too_many("queries")
    return ptr, elem, ld, nq


def scores(table: FlatTable, queries, dtype=None, out=None):
    """The scores (nq, n) of every record, (float(sum of code products) * query scale) * record scale [+ bias], in `dtype`
    (default float32) or into `out`."""
    torch = _t()
    ptr, elem, ld, nq = _queries(table, queries)
    if out is None:
        out = torch.empty((nq, table.n), dtype=dtype or torch.float32, device=table.device)
    elif (dtype is not None and out.dtype != dtype) or out.shape != (nq, table.n):
        raise ValueError(f"out must be ({nq}, {table.n}) of the asked dtype")
    optr, oelem, old = _rows(out, "out", table.device)[:3]
    lib = L.lib()
    size = lib.shine_flat_scores_workspace(nq, table.n, table.dim)
    ws = _workspace(size, table.device)
    L.check(lib.shine_flat_scores(table.device.index, C.byref(table._c), ptr, elem, nq, ld, optr, oelem, old,
                                  ws.data_ptr() if size else None, size, _stream(table.device)))
    return out


def adjust(scores, bias=None, allow=None, seen=None, repetition=None, frequency=None, presence=None, out=None):
    """Scores (nq, n) with penalties for shown records, biases and a filter, in this order, computed in float32:

    * seen (h,), (1, h) or (nq, h) int32, record ids, repeats counted, -1 skipped: a record met c > 0 times has its score
      divided by repetition[i] where positive and multiplied by it elsewhere, then frequency[i] * c + presence[i] taken
      off (float32 (nq,) each);
    * bias float32 (n,), (1, n) or (nq, n), added;
    * allow int32, (n + 31) // 32 words for all rows or for each: bit j % 32 of word j // 32 set where record j may be
      returned; the others' scores become -infinity.

    `out` may be `scores` itself.
    """
    torch = _t()
    ptr, elem, ld, nq, n = _rows(scores, "scores")
    if nq > MAX_ROWS:
        _too_many("scores")
    a = _adjustment(nq, n, scores.device, bias, allow, seen, repetition, frequency, presence)
    if out is None:
        out = torch.empty((nq, n), dtype=scores.dtype, device=scores.device)
    elif out.dtype != scores.dtype or out.shape != scores.shape:
        raise ValueError("out must have the scores' shape and dtype")
    optr, _, old = _rows(out, "out", scores.device)[:3]
    L.check(L.lib().shine_flat_adjust(scores.device.index, ptr, elem, nq, n, ld, C.byref(a), optr, old,
                                      _stream(scores.device)))
    return out


def topk(scores, k: int):
    """The k largest scores of every row in descending order, ties to the lower id: values (nq, k) and ids int32 (nq, k).
    -infinity and NaN are never returned: places without an answer hold id -1 and -infinity."""
    torch = _t()
    ptr, elem, ld, nq, n = _rows(scores, "scores")
    if nq > MAX_ROWS:
        _too_many("scores")
    if not 1 <= k <= MAX_K:
        raise ValueError(f"k must be in [1, {MAX_K}]")
    values = torch.empty((nq, k), dtype=scores.dtype, device=scores.device)
    ids = torch.empty((nq, k), dtype=torch.int32, device=scores.device)
    lib = L.lib()
    size = lib.shine_flat_topk_workspace(nq, n, k)
    ws = _workspace(size, scores.device)
    L.check(lib.shine_flat_topk(scores.device.index, ptr, elem, nq, n, ld, k, values.data_ptr(), ids.data_ptr(),
                                ws.data_ptr() if size else None, size, _stream(scores.device)))
    return values, ids


def search(table: FlatTable, queries, k: int, bias=None, allow=None, seen=None, repetition=None, frequency=None,
           presence=None):
    """topk(adjust(scores(table, queries), ...), k), bit for bit, without the score matrix: values float32 (nq, k) and ids
    int32 (nq, k)."""
    torch = _t()
    ptr, elem, ld, nq = _queries(table, queries)
    device = table.device
    if not 1 <= k <= MAX_K:
        raise ValueError(f"k must be in [1, {MAX_K}]")
    a = None
    if bias is not None or allow is not None or seen is not None or repetition is not None or frequency is not None or \
            presence is not None:
        a = C.byref(_adjustment(nq, table.n, device, bias, allow, seen, repetition, frequency, presence))
    values = torch.empty((nq, k), dtype=torch.float32, device=device)
    ids = torch.empty((nq, k), dtype=torch.int32, device=device)
    lib = L.lib()
    size = lib.shine_flat_search_workspace(nq, table.n, table.dim, k, a)
    ws = _workspace(size, device)
    L.check(lib.shine_flat_search(device.index, C.byref(table._c), ptr, elem, nq, ld, k, a, values.data_ptr(),
                                  ids.data_ptr(), ws.data_ptr() if size else None, size, _stream(device)))
    return values, ids
