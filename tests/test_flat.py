"""Flat scoring without a GPU: what its entries refuse, and the sizes they ask for.

The C entries look at their arguments before they touch a device, so every refusal is seen here; the pointers are made
up and never read.
"""
import ctypes as C

import pytest
import torch

from shine_amd import _lib as L
from shine_amd import flat

P = 0x10000  # aligned, never read


def table(**kw):
    t = dict(codes=P, scales=P, bias=None, n=100, dim=32)
    t.update(kw)
    return C.byref(L.FlatTable(t["codes"], t["scales"], t["bias"], t["n"], t["dim"], 0))


def adjustment(**kw):
    a = L.FlatAdjustment()
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


def refused(rc, text):
    assert rc == L.ERR_ARG
    assert text in L.lib().shine_last_error().decode()


def test_pitch_and_workspaces():
    lib = L.lib()
    for dim, pitch in ((1, 64), (64, 64), (65, 128), (96, 128), (200, 256), (16384, 16384)):
        assert lib.shine_flat_pitch(dim) == pitch == flat.code_pitch(dim)
    assert lib.shine_flat_scores_workspace(17, 1000, 96) >= 17 * 128 + 17 * 4
    assert lib.shine_flat_scores_workspace(7, 1 << 20, 300) >= 7 * 320 + 7 * 4
    assert lib.shine_flat_search_workspace(7, 1000, 96, 10, None) >= 7 * 128 + 7 * 4


def test_quantize_refusals():
    f = L.lib().shine_flat_quantize
    refused(f(0, P, 0, 10, 0, 8, P, P, None, None), "dim")
    refused(f(0, P, 0, 10, 16385, 16385, P, P, None, None), "dim")
    refused(f(0, P, 2, 10, 8, 8, P, P, None, None), "element type")
    refused(f(0, None, 0, 10, 8, 8, P, P, None, None), "NULL")
    refused(f(0, P, 0, 10, 8, 7, P, P, None, None), "stride")
    refused(f(0, P + 2, 0, 10, 8, 8, P, P, None, None), "aligned")
    refused(f(0, P, 0, 10, 8, 8, None, P, None, None), "NULL")
    refused(f(0, P, 0, 10, 8, 8, P, None, None, None), "NULL")
    refused(f(0, P, 0, 10, 8, 8, P + 4, P, None, None), "aligned")
    refused(f(0, P, 0, 10, 8, 8, P, P + 1, None, None), "aligned")
    assert f(0, None, 0, 0, 8, 8, None, None, None, None) == L.OK  # no rows: nothing to do, no device needed


def test_scores_refusals():
    f = L.lib().shine_flat_scores
    big = 1 << 40
    refused(f(0, None, P, 0, 4, 32, P, 0, 100, P, big, None), "table")
    refused(f(0, table(dim=0), P, 0, 4, 32, P, 0, 100, P, big, None), "dim")
    refused(f(0, table(n=(1 << 30) + 1), P, 0, 4, 32, P, 0, 1 << 31, P, big, None), "2^30")
    refused(f(0, table(codes=None), P, 0, 4, 32, P, 0, 100, P, big, None), "NULL")
    refused(f(0, table(codes=P + 16), P, 0, 4, 32, P, 0, 100, P, big, None), "64-byte")
    refused(f(0, table(), P, 3, 4, 32, P, 0, 100, P, big, None), "element type")
    refused(f(0, table(), None, 0, 4, 32, P, 0, 100, P, big, None), "NULL")
    refused(f(0, table(), P, 0, 4, 31, P, 0, 100, P, big, None), "stride")
    refused(f(0, table(), P, 0, 4, 32, P, 2, 100, P, big, None), "element type")
    refused(f(0, table(), P, 0, 4, 32, P, 0, 99, P, big, None), "stride")
    refused(f(0, table(), P, 0, 17, 32, P, 0, 100, None, big, None), "workspace")
    refused(f(0, table(), P, 0, 17, 32, P, 0, 100, P + 128, big, None), "workspace")
    refused(f(0, table(), P, 0, 17, 32, P, 0, 100, P, 100, None), "workspace")
    assert f(0, table(), None, 0, 0, 32, None, 0, 100, None, 0, None) == L.OK
    assert f(0, table(n=0, codes=None, scales=None), P, 0, 4, 32, None, 0, 0, None, 0, None) == L.OK


def test_adjust_refusals():
    f = L.lib().shine_flat_adjust
    refused(f(0, P, 0, 4, 100, 100, None, P, 100, None), "adjustment")
    refused(f(0, P, 0, 4, (1 << 30) + 1, 1 << 31, adjustment(), P, 1 << 31, None), "2^30")
    refused(f(0, P, 4, 4, 100, 100, adjustment(), P, 100, None), "element type")
    refused(f(0, P, 0, 4, 100, 99, adjustment(), P, 100, None), "stride")
    refused(f(0, P, 0, 4, 100, 100, adjustment(), P, 99, None), "stride")
    refused(f(0, P, 0, 4, 100, 100, adjustment(), None, 100, None), "NULL")
    refused(f(0, P, 0, 4, 100, 100, adjustment(bias=P, bias_ld=99), P, 100, None), "bias row stride")
    refused(f(0, P, 0, 4, 100, 100, adjustment(allow=P, allow_ld=3), P, 100, None), "allow row stride")
    refused(f(0, P, 0, 4, 100, 100, adjustment(seen_n=3), P, 100, None), "seen is NULL")
    refused(f(0, P, 0, 4, 100, 100, adjustment(seen=P, seen_n=3, seen_ld=2), P, 100, None), "seen row stride")
    refused(f(0, P, 0, 4, 100, 100, adjustment(seen=P, seen_n=65536, seen_ld=65536), P, 100, None), "65535")
    refused(f(0, P, 0, 4, 100, 100, adjustment(bias=P + 2), P, 100, None), "4-byte")
    assert f(0, None, 0, 0, 100, 100, adjustment(), None, 100, None) == L.OK
    assert f(0, None, 0, 4, 0, 0, adjustment(), None, 0, None) == L.OK


def test_topk_refusals():
    f = L.lib().shine_flat_topk
    for k in (0, 257):
        refused(f(0, P, 0, 4, 100, 100, k, P, P, None, 0, None), "k must")
    refused(f(0, P, 0, 4, (1 << 30) + 1, 1 << 31, 10, P, P, None, 0, None), "2^30")
    refused(f(0, P, 7, 4, 100, 100, 10, P, P, None, 0, None), "element type")
    refused(f(0, P, 0, 4, 100, 99, 10, P, P, None, 0, None), "stride")
    refused(f(0, None, 0, 4, 100, 100, 10, P, P, None, 0, None), "NULL")
    refused(f(0, P, 0, 4, 100, 100, 10, None, P, None, 0, None), "NULL")
    refused(f(0, P, 0, 4, 100, 100, 10, P, None, None, 0, None), "NULL")
    refused(f(0, P, 0, 4, 100, 100, 10, P, P + 2, None, 0, None), "aligned")
    need = L.lib().shine_flat_topk_workspace(1, 1_000_000, 10)
    assert need > 0
    refused(f(0, P, 0, 1, 1_000_000, 1_000_000, 10, P, P, None, need, None), "workspace")
    refused(f(0, P, 0, 1, 1_000_000, 1_000_000, 10, P, P, P, need - 1, None), "workspace")
    assert f(0, None, 0, 0, 100, 100, 10, None, None, None, 0, None) == L.OK


def test_search_refusals():
    f = L.lib().shine_flat_search
    big = 1 << 40
    refused(f(0, None, P, 0, 4, 32, 10, None, P, P, P, big, None), "table")
    refused(f(0, table(), P, 0, 4, 32, 0, None, P, P, P, big, None), "k must")
    refused(f(0, table(), P, 0, 4, 32, 257, None, P, P, P, big, None), "k must")
    refused(f(0, table(), P, 0, 4, 31, 10, None, P, P, P, big, None), "stride")
    refused(f(0, table(), P, 0, 4, 32, 10, adjustment(allow=P, allow_ld=3), P, P, P, big, None), "allow row stride")
    refused(f(0, table(), P, 0, 4, 32, 10, None, None, P, P, big, None), "NULL")
    refused(f(0, table(), P, 0, 4, 32, 10, None, P, P + 2, P, big, None), "aligned")
    refused(f(0, table(), P, 0, 4, 32, 10, None, P, P, None, big, None), "workspace")
    need = L.lib().shine_flat_search_workspace(4, 100, 32, 10, None)
    refused(f(0, table(), P, 0, 4, 32, 10, None, P, P, P, need - 1, None), "workspace")
    assert f(0, table(), None, 0, 0, 32, 10, None, None, None, None, 0, None) == L.OK


def test_python_refuses_what_is_no_gpu_row_tensor():
    for bad in ([[1.0]], torch.zeros(4), torch.zeros(2, 2, 2)):
        with pytest.raises(ValueError, match="2-D"):
            flat.quantize_rows(bad)
    with pytest.raises(ValueError, match="float32"):
        flat.quantize_rows(torch.zeros(2, 2, dtype=torch.float64))
    with pytest.raises(ValueError, match="on a GPU"):
        flat.topk(torch.zeros(2, 2), 1)
    with pytest.raises(ValueError, match="metric"):
        flat.FlatTable(torch.zeros(2, 2), metric="cosine")
    with pytest.raises(ValueError, match="FlatTable"):
        flat.search(torch.zeros(2, 2), torch.zeros(2, 2), 1)


def test_adjust_refuses_rows_that_overlap():
    f = L.lib().shine_flat_adjust
    for out, ld, out_ld in ((P + 4, 100, 100), (P, 100, 101), (P + 396, 100, 100), (P - 396, 100, 100), (P + 99 * 4, 250, 250),
                            (P + (250 + 151) * 4, 250, 250), (P + 1000, 100, 300)):
        refused(f(0, P, 0, 4, 100, ld, adjustment(), out, out_ld, None), "overlaps")
    refused(f(0, P, 0, 1, 100, 100, adjustment(), P + 4, 100, None), "overlaps")


def test_a_history_of_stride_0_is_shared_by_all_rows():
    """accepted as a shared bias or mask is: what is refused next is the missing workspace, or the overlap"""
    a = dict(seen=P, seen_n=3, seen_ld=0)
    refused(L.lib().shine_flat_search(0, table(), P, 0, 4, 32, 10, adjustment(**a), P, P, None, 1 << 40, None), "workspace")
    refused(L.lib().shine_flat_adjust(0, P, 0, 4, 100, 100, adjustment(**a), P + 4, 100, None), "overlaps")


def test_search_workspace_of_what_search_refuses():
    """sizes beyond the limits have no plan: 0, and search refuses them before it asks for a workspace"""
    f = L.lib().shine_flat_search_workspace
    assert f(17, 1 << 30, 96, 10, None) > 0
    for n, dim, k in (((1 << 30) + 1, 96, 10), (1 << 60, 96, 10), ((1 << 64) - 1, 96, 10), (1000, 0, 10), (1000, 16385, 10),
                      (1000, 2 ** 32 - 1, 10), (1000, 96, 0), (1000, 96, 257)):
        assert f(17, n, dim, k, None) == 0


def test_a_tables_parts_stay():
    """the C table names their memory: replacing one would let calls read what is no longer held"""
    t = flat.FlatTable.__new__(flat.FlatTable)
    parts = dict(codes=torch.zeros((3, 64), dtype=torch.int8), scales=torch.ones(3), bias=torch.zeros(3), n=3, dim=2, metric="l2",
                 device=torch.device("cpu"), _c=None)
    for name, part in parts.items():
        setattr(t, name, part)
    for name, part in parts.items():
        with pytest.raises(AttributeError, match="replaced"):
            setattr(t, name, part.clone() if isinstance(part, torch.Tensor) else object())
        with pytest.raises(AttributeError, match="taken away"):
            delattr(t, name)
        assert getattr(t, name) is part
    t.bias += 1  # in place
    t.name = "a table's own name"
    del t.name
    assert t.bias.tolist() == [1, 1, 1]
