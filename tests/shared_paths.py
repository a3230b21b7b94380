"""Calls of kvcache.decode_shared that reach each of its kernels' instances: the tables are wide enough for the path,
the lengths in them short."""
import ctypes

import torch

WHOLE, ROWS, BOTH, LAST, APART = range(5)  # out[0] of tallax_testing_shared_plan
NAMES = ("whole", "rows", "both", "last", "apart")
PAGE = 16


class Case:
    def __init__(self, path, rg, mt, dtype, dim, batch, prompts, queries, group, kv_heads, prefix_pages, own_pages, page=PAGE):
        self.path, self.rg, self.mt, self.dtype, self.dim = path, rg, mt, dtype, dim
        self.batch, self.prompts, self.queries, self.group, self.kv_heads = batch, prompts, queries, group, kv_heads
        self.prefix_pages, self.own_pages, self.page = prefix_pages, own_pages, page

    def __repr__(self):
        t = "bf16" if self.dtype == torch.bfloat16 else "f32"
        return (f"{NAMES[self.path]}-rg{self.rg}-mt{self.mt}-{t}-{self.dim}-{self.batch}x{self.queries}x{self.group}"
                f"x{self.kv_heads}-{self.prompts}-{self.prefix_pages}-{self.own_pages}" + (f"-p{self.page}" if self.page != PAGE else ""))

    def plan(self):
        """What the library makes of it."""
        from tallax_amd import _lib
        n = self.kv_heads * self.page * self.dim
        strides = {f"{x}_stride_{y}": s for x in "kv" for y, s in (("page", n), ("head", self.page * self.dim), ("slot", self.dim))}
        c = _lib.KvCache(k=4096, v=4096, dtype=_lib.BF16 if self.dtype == torch.bfloat16 else _lib.F32, dim=self.dim,
                         pages=4096, kv_heads=self.kv_heads, page_size=self.page, block_table=4096, batch=self.batch,
                         table_width=self.own_pages, **strides)
        out = (ctypes.c_int32 * 6)()
        _lib.check(_lib.LIB.tallax_testing_shared_plan(ctypes.byref(c), self.prompts, self.prefix_pages, self.queries,
                                                       self.group * self.kv_heads, -1, -1, out), "plan")
        return list(out)


def cases():
    r = []
    for dtype in (torch.bfloat16, torch.float32):
        f32 = dtype == torch.float32
        for dim in (40, 64, 80, 128, 192, 256):
            add = lambda path, rg, mt, *a: r.append(Case(path, rg, mt, dtype, dim, *a))  # noqa: E731,B023
            two = f32 or dim <= 128  # two sixteens of rows to a workgroup
            whole = dim in (64, 128, 256)  # no elements past dim in an instance
            narrow = 4 if f32 and dim > 128 else 2
            # few rows, of one query and of several, in one sixteen and in two
            if whole:
                add(ROWS, 0, 1, 2, 1, 1, 4, 2, 60, 60)
            add(ROWS, 0, 1, 4, 2, 3, 2, 2, 60, 60)
            add(ROWS, 0, 1, 1, 1, 13, 1, 3, 130, 1)
            if two:
                add(ROWS, 0, 2, 4, 1, 1, 8, 2, 60, 60)
                add(ROWS, 0, 2, 4, 2, 5, 3, 2, 60, 60)
            # tiles and own slots in one launch
            add(BOTH, narrow, 1, 39, 3, 1, 3, 2, 130, 60)
            if whole:
                add(BOTH, 4, 1, 24, 1, 1, 5, 2, 130, 10)
            add(BOTH, 4, 1, 24, 1, 3, 5, 2, 60, 130)
            if two:
                add(BOTH, 4, 2, 24, 1, 5, 4, 2, 130, 60)
                add(BOTH, narrow, 2, 9, 3, 5, 4, 2, 130, 60)
            else:
                add(BOTH, 4, 1, 24, 1, 5, 4, 2, 130, 60)  # two workgroups share a sequence's rows
                add(BOTH, 2, 1, 9, 3, 5, 4, 2, 130, 60)
            # tiles, then own slots in one chunk each, whose workgroups make the outputs
            if whole:
                add(LAST, 4, 1, 132, 1, 1, 3, 2, 60, 60)
            add(LAST, 4, 1, 132, 1, 3, 2, 2, 60, 60)
            if two:
                add(LAST, 4, 2, 132, 1, 5, 4, 2, 130, 10)
                add(LAST, narrow, 2, 129, 43, 5, 4, 2, 60, 60)
                add(LAST, 4, 2, 130, 2, 1, 18, 2, 130, 20)  # one query
            else:
                add(LAST, 4, 1, 132, 1, 5, 4, 2, 60, 10)
            add(LAST, narrow, 1, 132, 11, 1, 4, 2, 10, 130)
            # tiles, then the decode kernel, then the join
            if whole:
                add(APART, narrow, 1, 60, 10, 1, 6, 4, 60000, 10)
            add(APART, narrow, 1, 60, 10, 1, 6, 4, 60000, 60)
            if not whole:
                add(APART, 4, 1, 50, 1, 3, 3, 5, 60000, 10)
                continue
            add(APART, 4, 1, 50, 1, 3, 3, 5, 60000, 60)
            if two:
                add(APART, 4, 2, 50, 1, 6, 3, 5, 60000, 10)
                add(APART, 4, 2, 40, 1, 1, 20, 5, 60000, 60)
            if not f32 and dim == 128:
                add(APART, 2, 1, 210, 70, 3, 4, 8, 60, 10)
    return r


def cases_of_pages():
    """Pages of one slot, of sizes that are no power of two and end inside tiles, and of more than a chunk."""
    r = []
    for dtype in (torch.bfloat16, torch.float32):
        for dim in (64, 128, 192):
            f32 = dtype == torch.float32
            mt, narrow = (2 if f32 or dim <= 128 else 1), (4 if f32 and dim > 128 else 2)
            for page in (1, 7, 24, 100, 1000):
                for path, rg, m, calls, slots, own in ((ROWS, 0, 1, (4, 2, 3, 2, 2), 1000, 1000), (BOTH, 4, 1, (24, 1, 3, 5, 2), 2100, 1000),
                                                       (LAST, 4, mt, (132, 1, 5, 4, 2), 2000, 160), (APART, narrow, 1, (60, 10, 1, 6, 4), 960000, 200)):
                    r.append(Case(path, rg, m, dtype, dim, *calls, -(-slots // page), -(-own // page), page))
    return r


def cases_of_dims():
    """Dims from the smallest on that leave most of a kernel's instance empty, or all but eight elements of it full."""
    r = []
    for dtype in (torch.bfloat16, torch.float32):
        for dim in (8, 24, 56, 72, 104, 136, 248):
            f32 = dtype == torch.float32
            mt, narrow = (2 if f32 or dim <= 128 else 1), (4 if f32 and dim > 128 else 2)
            r.append(Case(ROWS, 0, 1, dtype, dim, 4, 2, 3, 2, 2, 140, 60))
            r.append(Case(BOTH, 4, 1, dtype, dim, 24, 1, 3, 5, 2, 200, 60))
            r.append(Case(BOTH, narrow, 1, dtype, dim, 39, 3, 1, 3, 2, 200, 60))
            r.append(Case(LAST, 4, mt, dtype, dim, 132, 1, 5, 4, 2, 200, 10))
            r.append(Case(APART, narrow, 1, dtype, dim, 60, 10, 1, 6, 4, 60000, 60))
    return r


def cases_of_many_rows():
    """The most rows of a sequence's kv head."""
    r = []
    for dtype in (torch.bfloat16, torch.float32):
        r.append(Case(BOTH, 4, 2, dtype, 64, 1, 1, 1024, 4, 1, 200, 90))
        r.append(Case(LAST, 4, 2, dtype, 64, 2, 1, 1024, 4, 1, 200, 90))
    return r
