"""Host: the calls of tests/shared_paths.py are planned as the tests of their kernels need them."""
import ctypes

import torch

from tests import shared_paths as S
from tests.test_serving_host import _cache


def test_each_case_takes_its_path():
    reached = set()
    for c in S.cases():
        path, rg, mt, row_groups, chunks, own_chunks = c.plan()
        assert (path, rg, mt) == (c.path, c.rg, c.mt), (c, path, rg, mt)
        assert row_groups == (1 if path == S.ROWS else -(-c.queries * c.group // (16 * mt))) and chunks >= 1
        dims = 64 if c.dim <= 64 else 128 if c.dim <= 128 else 256
        reached.add((path, rg, mt, c.dtype, dims, c.queries > 1 or path == S.BOTH))
        reached.add((path, c.dtype, dims, own_chunks > 1))
    for c in S.cases_of_pages() + S.cases_of_dims() + S.cases_of_many_rows():
        assert c.plan()[:3] == [c.path, c.rg, c.mt], (c, c.plan())
    for dtype in (torch.bfloat16, torch.float32):
        for dims in (64, 128, 256):
            sixteens = (1, 2) if dtype == torch.float32 or dims <= 128 else (1,)
            groups = (4,) if dtype == torch.float32 and dims > 128 else (2, 4)
            for mt in sixteens:
                for many in (False, True):
                    assert (S.ROWS, 0, mt, dtype, dims, many) in reached
                    assert any((S.LAST, rg, mt, dtype, dims, many) in reached for rg in groups)
                for rg in groups:
                    assert (S.BOTH, rg, mt, dtype, dims, True) in reached
                    assert any((S.LAST, rg, m, dtype, dims, many) in reached for m in sixteens for many in (False, True))
                    assert any((S.APART, rg, m, dtype, dims, many) in reached for m in sixteens for many in (False, True))
            for many in (False, True):
                for path in (S.ROWS, S.BOTH, S.APART):
                    assert (path, dtype, dims, many) in reached


def test_the_plan_is_refused_where_the_call_is():
    from tallax_amd import _lib
    out = (ctypes.c_int32 * 6)()
    plan = _lib.LIB.tallax_testing_shared_plan
    good = dict(prefixes=1, width=4, queries=1, heads=4, max_prefix=-1, max_len=-1)
    c = _cache()
    assert plan(ctypes.byref(c), *good.values(), out) == _lib.OK and out[0] == S.WHOLE
    assert plan(ctypes.byref(c), *good.values(), None) == _lib.INVALID_ARGUMENT
    for over in (dict(prefixes=2), dict(prefixes=0), dict(width=-1), dict(queries=0), dict(queries=2000), dict(heads=3)):
        assert plan(ctypes.byref(c), *{**good, **over}.values(), out) == _lib.INVALID_ARGUMENT, over
    assert plan(ctypes.byref(_cache(dim=60)), *good.values(), out) == _lib.INVALID_ARGUMENT
