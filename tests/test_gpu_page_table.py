"""The bookkeeping of a cache in pages (psx_b200_extend_pages, fork_pages, release_pages, compact_pages) against a restatement that
takes rows one after the other: whole numbers and copied bytes, so everything is equal."""
import ctypes as C

import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx

pytestmark = pytest.mark.gpu


class Book:
    """A page table and pools as lists and arrays."""

    def __init__(self, rows, max_pages, num_pages, size, pools):
        self.table = [[-1] * max_pages for _ in range(rows)]
        self.lengths, self.references, self.size, self.most, self.pools = [0] * rows, [0] * num_pages, size, max_pages, pools

    def pages(self, row, length=None):
        return self.table[row][:-(-(self.lengths[row] if length is None else length) // self.size)]

    def extend(self, added):
        size, status = self.size, []
        free = [p for p, n in enumerate(self.references) if n == 0]
        held, before = list(self.references), list(self.lengths)
        fits = [n >= 0 and before[b] + n <= self.most * size for b, n in enumerate(added)]
        going = {}
        for b, n in enumerate(added):
            if fits[b] and n > 0 and before[b] % size:
                going.setdefault(self.table[b][before[b] // size], []).append(b)
        asked = 0
        for b, n in enumerate(added):
            if not fits[b]:
                status.append(psx.ROW_BAD_OFFSETS if n < 0 else psx.ROW_CACHE_FULL)
                continue
            entries = list(range(-(-before[b] // size), -(-(before[b] + n) // size)))
            old = self.table[b][before[b] // size] if n > 0 and before[b] % size else None
            parts = old is not None and held[old] > 1 and not (len(going[old]) == held[old] and going[old][-1] == b)
            if parts:
                entries.insert(0, before[b] // size)
            asked += len(entries)
            if entries and asked > sum(1 for x in held if x == 0):
                status.append(psx.ROW_CACHE_FULL)
                continue
            for i, at in enumerate(entries):
                page = free.pop(0)
                self.references[page] = 1
                if parts and i == 0:
                    self.references[old] -= 1
                    for pool in self.pools:
                        pool[page, :, :before[b] % size] = pool[old, :, :before[b] % size]
                self.table[b][at] = page
            self.lengths[b] = before[b] + n
            status.append(0)
        return status

    def fork(self, parents):
        beams = len(parents[0])
        rows = [(self.pages(b), self.lengths[b]) for b in range(len(self.table))]
        for g, chosen in enumerate(parents):
            for j, p in enumerate(chosen):
                if not 0 <= p < beams:
                    continue
                b, (pages, length) = g * beams + j, rows[g * beams + p]
                for x in rows[b][0]:
                    self.references[x] -= 1
                for x in pages:
                    self.references[x] += 1
                self.table[b][:len(pages)], self.lengths[b] = pages, length

    def release(self, keep):
        for b in range(len(self.table)):
            kept = 0 if keep is None else min(max(keep[b], 0), self.lengths[b])
            for x in self.pages(b)[-(-kept // self.size):]:
                self.references[x] -= 1
            self.lengths[b] = kept

    def compact(self):
        used = sum(1 for n in self.references if n)
        movers, goals = [p for p in range(used, len(self.references)) if self.references[p]], [p for p in range(used) if not self.references[p]]
        goal = dict(zip(movers, goals))
        for a, b in goal.items():
            self.references[b], self.references[a] = self.references[a], 0
            for pool in self.pools:
                pool[b] = pool[a]
        for b in range(len(self.table)):
            self.table[b][:len(self.pages(b))] = [goal.get(p, p) for p in self.pages(b)]
        return used

    def check(self, table, pools):
        import torch
        torch.cuda.synchronize()
        assert table.lengths.tolist() == self.lengths
        assert table.references.tolist() == self.references
        found = table.pages.tolist()
        for b in range(len(self.table)):
            assert found[b][:len(self.pages(b))] == self.pages(b), b
        for mine, theirs in zip(self.pools, pools):
            assert (theirs.cpu().numpy() == mine).all()


def _pools(rng, num_pages, size, shapes):
    import torch
    pools = []
    for heads, dims, kind in shapes:
        x = rng.randint(0, 256, (num_pages, heads, size, dims * np.dtype(kind).itemsize)).astype(np.uint8).view(kind)
        pools.append(np.ascontiguousarray(x if kind != np.float32 else rng.randn(num_pages, heads, size, dims).astype(np.float32)))
    return pools, [torch.from_numpy(p.copy()).cuda() for p in pools]


def _whole(values, kind="int64"):
    import torch
    return torch.tensor(values, dtype=getattr(torch, kind), device="cuda")


def _both(rng, rows, max_pages, num_pages, size, shapes=((2, 8, np.float32), (1, 3, np.uint8))):
    mine, theirs = _pools(rng, num_pages, size, shapes)
    return Book(rows, max_pages, num_pages, size, mine), psx.PageTable.empty(rows, max_pages, num_pages, size), theirs


@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("groups,beams,num_pages,seed", [(1, 1, 7, 0), (1, 4, 40, 1), (5, 3, 60, 2), (2, 8, 4101, 3), (7, 5, 30, 4), (1, 64, 200, 5)])
def test_a_run_of_calls(size, groups, beams, num_pages, seed):
    rng = np.random.RandomState(seed)
    rows, max_pages = groups * beams, 9
    book, table, pools = _both(rng, rows, max_pages, num_pages, size, ((2, 8, np.float32), (1, 3, np.uint8), (3, 5, np.int16), (1, 8, np.uint8)))
    ctx = gh.ctx()
    for step in range(40):
        call = rng.randint(0, 10) if step > 2 else 0
        if call < 5:
            top = rng.choice([1, 2, size, 3 * size])
            added = rng.randint(0, top + 1, rows) * (rng.rand(rows) < 0.8)
            if rng.rand() < 0.1:
                added[rng.randint(rows)] = -1
            status = ctx.extend_pages(table, _whole(added), pools)
            assert status.tolist() == book.extend(added.tolist())
        elif call < 7:
            parents = rng.randint(-1, beams + 1, (groups, beams))
            ctx.fork_pages(table, _whole(parents))
            book.fork(parents.tolist())
        elif call < 9:
            keep = rng.randint(-2, max_pages * size + 1, rows)
            ctx.release_pages(table, _whole(keep))
            book.release(keep.tolist())
        else:
            assert int(ctx.compact_pages(table, pools)) == book.compact()
        book.check(table, pools)
    ctx.release_pages(table)
    book.release(None)
    book.check(table, pools)
    assert not table.references.any() and not table.lengths.any()


def test_rows_that_part():
    # one prompt, four beams: three copies of the last page, and the last beam keeps it; with a fifth holder, four copies
    rng = np.random.RandomState(0)
    for beams, going in ((4, [1, 1, 1, 1]), (5, [1, 1, 1, 1, 0]), (4, [0, 1, 1, 0])):
        book, table, pools = _both(rng, beams, 4, 20, 16)
        ctx = gh.ctx()
        for call, mine in ((lambda: ctx.extend_pages(table, _whole([37] + [0] * (beams - 1)), pools), lambda: book.extend([37] + [0] * (beams - 1))),
                           (lambda: ctx.fork_pages(table, _whole([[0] * beams])), lambda: book.fork([[0] * beams])),
                           (lambda: ctx.extend_pages(table, _whole(going), pools), lambda: book.extend(going))):
            call(), mine()
            book.check(table, pools)
        held = table.references.tolist()
        assert held[:2] == [beams, beams]
        assert sorted(held[2:])[-sum(going) - 1:] == [0, 1, 1, 1, 1] if beams == sum(going) else [1] * sum(going) + [beams - sum(going)]


def test_rows_for_which_there_are_no_pages():
    rng = np.random.RandomState(0)
    book, table, pools = _both(rng, 5, 3, 4, 16)
    for added in ([16, 17, 0, 30, 1], [0, 0, 0, 16, 16], [0, 0, 0, 1, 0], [1, 31, 0, 0, 0], [0, 15, 0, 0, 0], [100, 2 ** 62, -2 ** 62, 0, 0]):
        status = gh.ctx().extend_pages(table, _whole(added), pools).tolist()
        assert status == book.extend(added)
        book.check(table, pools)


def test_numbers_that_make_no_sense_are_left_alone():
    import torch
    ctx = gh.ctx()
    table = psx.PageTable(_whole([[5, 0], [1, 9], [-3, 0], [0, 1], [2, 0]], "int32"), _whole([3, 20, 1, -1, 33]), _whole([1, 1, 1, 0, 0, 0], "int32"), 16)
    before = [x.clone() for x in (table.pages, table.lengths)]
    assert ctx.extend_pages(table, _whole([1, 1, 1, 1, 1])).tolist()[1:] == [65, 65, 65, 65]  # (page 9 of 6, page -3, lengths out of range)
    torch.cuda.synchronize()
    assert (table.pages == before[0]).all() and (table.lengths[1:] == before[1][1:]).all()
    # pages that are none lose nothing; a length beyond the row's two entries counts as all of them, so the last row gives back pages 2 and 0, the
    # second one page 1, and the first one page 5, which nobody had counted
    ctx.release_pages(table)
    assert table.lengths.tolist()[:3] == [0, 0, 0] and table.lengths.tolist()[4] == 0 and table.references.tolist() == [0, 0, 0, 0, 0, -1]


@pytest.mark.parametrize("num_pages", [1, 2, 3, 4095, 4096, 4097, 70001])
def test_many_pages(num_pages):
    rng = np.random.RandomState(num_pages)
    size, rows, max_pages = 16, 7, num_pages
    book, table, pools = _both(rng, rows, max_pages, num_pages, size, ((1, 1, np.uint8),))
    ctx = gh.ctx()
    share = num_pages // rows
    for step in range(4):
        added = [int(x) for x in rng.randint(0, max(2, share * size // 2), rows)]
        assert ctx.extend_pages(table, _whole(added), pools).tolist() == book.extend(added)
        keep = [int(x) for x in rng.randint(0, max(2, share * size), rows)]
        ctx.release_pages(table, _whole(keep))
        book.release(keep)
        if step % 2:
            assert int(ctx.compact_pages(table, pools)) == book.compact()
        book.check(table, pools)


def test_references_that_start_anywhere():
    import torch
    rng = np.random.RandomState(9)
    for shift in (1, 2, 3):
        book, _, pools = _both(rng, 3, 6, 5000 + shift, 16, ((1, 1, np.uint8),))
        table = psx.PageTable(torch.full((3, 6), -1, dtype=torch.int32, device="cuda"), _whole([0, 0, 0]), _whole([9] * shift + [0] * (5000 + shift), "int32")[shift:], 16)
        ctx = gh.ctx()
        for added in ([40, 3, 0], [1, 60, 17]):
            assert ctx.extend_pages(table, _whole(added), pools).tolist() == book.extend(added)
        ctx.release_pages(table, _whole([0, 30, 17])), book.release([0, 30, 17])
        assert int(ctx.compact_pages(table, pools)) == book.compact()
        book.check(table, pools)


def test_as_many_rows_as_there_may_be():
    rng = np.random.RandomState(1)
    book, table, pools = _both(rng, 4096, 2, 9000, 16, ((1, 4, np.uint8),))
    ctx = gh.ctx()
    added = rng.randint(0, 20, 4096).tolist()
    assert ctx.extend_pages(table, _whole(added), pools).tolist() == book.extend(added)
    parents = rng.randint(0, 64, (64, 64))
    ctx.fork_pages(table, _whole(parents)), book.fork(parents.tolist())
    assert ctx.extend_pages(table, _whole([1] * 4096), pools).tolist() == book.extend([1] * 4096)
    book.check(table, pools)


def test_more_pools_than_a_launch_takes():
    import torch
    rng = np.random.RandomState(2)
    book, table, pools = _both(rng, 2, 3, 12, 16, ((1, 4, np.uint8),) * 70)
    ctx = gh.ctx()
    for added, parents in (([20, 0], [[0, 0]]), ([1, 1], [[1, 1]]), ([3, 0], [[0, 1]])):
        assert ctx.extend_pages(table, _whole(added), pools).tolist() == book.extend(added)
        ctx.fork_pages(table, _whole(parents)), book.fork(parents)
    ctx.release_pages(table, _whole([0, 40])), book.release([0, 40])
    assert int(ctx.compact_pages(table, pools)) == book.compact()
    book.check(table, pools)


def test_pages_larger_than_a_piece_and_no_pools():
    rng = np.random.RandomState(3)
    book, table, pools = _both(rng, 3, 8, 24, 128, ((4, 96, np.float32), (1, 7, np.uint8)))
    ctx = gh.ctx()
    for added in ([1000, 500, 300], [0, 100, 700]):
        assert ctx.extend_pages(table, _whole(added), pools).tolist() == book.extend(added)
    ctx.release_pages(table, _whole([0, 1000, 1000])), book.release([0, 1000, 1000])
    assert int(ctx.compact_pages(table, pools)) == book.compact()
    book.check(table, pools)
    empty = psx.PageTable.empty(2, 2, 5, 16)
    assert ctx.extend_pages(empty, _whole([17, 5])).tolist() == [0, 0]
    ctx.release_pages(empty, _whole([0, 5]))
    assert int(ctx.compact_pages(empty, [])) == 1 and empty.pages[1, 0] == 0
    none = psx.PageTable.empty(0, 2, 5, 16)
    assert ctx.extend_pages(none, _whole([])).tolist() == [] and int(ctx.compact_pages(none, [])) == 0
    ctx.release_pages(none)


def test_captured_calls_use_what_the_replay_finds():
    import torch
    ctx = psx.Context(0)
    rng = np.random.RandomState(4)
    book, table, pools = _both(rng, 6, 6, 40, 16)
    added, parents, keep = _whole([0] * 6), _whole([[0, 1, 2], [0, 1, 2]]), _whole([96] * 6)

    def step():
        ctx.release_pages(table, keep)
        ctx.fork_pages(table, parents)
        status = ctx.extend_pages(table, added, pools)
        return status, ctx.compact_pages(table, pools)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        status, used = step()
    for _ in range(8):
        kept, chosen, more = rng.randint(0, 96, 6), rng.randint(0, 3, (2, 3)), rng.randint(0, 25, 6)
        keep.copy_(torch.from_numpy(kept)), parents.copy_(torch.from_numpy(chosen)), added.copy_(torch.from_numpy(more))
        graph.replay()
        torch.cuda.synchronize()
        book.release(kept.tolist()), book.fork(chosen.tolist())
        assert status.tolist() == book.extend(more.tolist()) and int(used) == book.compact()
        book.check(table, pools)


def test_another_stream():
    import torch
    rng = np.random.RandomState(5)
    book, table, pools = _both(rng, 4, 4, 30, 16)
    ctx, stream = gh.ctx(), torch.cuda.Stream()
    added, parents = _whole([20, 0, 3, 0]), _whole([[0, 0, 2, 2]])
    stream.wait_stream(torch.cuda.current_stream())
    for given in (None, stream.cuda_stream):
        with torch.cuda.stream(stream if given is None else torch.cuda.current_stream()):
            ctx.extend_pages(table, added, pools, stream=given)
            ctx.fork_pages(table, parents, stream=given)
        book.extend([20, 0, 3, 0]), book.fork([[0, 0, 2, 2]])
        stream.synchronize()
        book.check(table, pools)


def test_refusals():
    import torch
    ctx, table = gh.ctx(), psx.PageTable.empty(4, 4, 8, 16)
    pool, ones = torch.zeros(8, 2, 16, 4, device="cuda"), _whole([1] * 4)
    for bad in (pool[:7], pool.transpose(1, 2), pool[:, 0], pool.cpu()):
        with pytest.raises(ValueError):
            ctx.extend_pages(table, ones, [bad])
        with pytest.raises(ValueError):
            ctx.compact_pages(table, [bad])
    for bad in (ones[:3], ones.int(), ones.cpu(), torch.ones(8, dtype=torch.int64, device="cuda")[::2]):
        with pytest.raises(ValueError):
            ctx.extend_pages(table, bad)
        with pytest.raises(ValueError):
            ctx.release_pages(table, bad)
    for bad in (ones, ones.view(2, 2).int(), _whole([[0, 1]]), ones.view(2, 2).t()):
        with pytest.raises(ValueError):
            ctx.fork_pages(table, bad)
    for bad in (dict(page_size=8), dict(page_size=256), dict(page_size=48)):
        with pytest.raises(psx.PsxError) as e:
            ctx.extend_pages(psx.PageTable.empty(4, 4, 8, **bad), ones)
        assert e.value.status == psx.ERR_UNSUPPORTED
    with pytest.raises(psx.PsxError) as e:
        ctx.release_pages(psx.PageTable.empty(4097, 1, 1, 16))
    assert e.value.status == psx.ERR_UNSUPPORTED
    with pytest.raises(psx.PsxError) as e:
        ctx.fork_pages(psx.PageTable.empty(65, 1, 1, 16), torch.zeros(1, 65, dtype=torch.int64, device="cuda"))
    assert e.value.status == psx.ERR_UNSUPPORTED
    wide = torch.zeros(8 * 128 + 4, device="cuda")
    for pools in ([pool, pool], [wide[:1024].view(8, 2, 16, 4), wide[4:1028].view(8, 2, 16, 4)]):
        for call in (lambda: ctx.extend_pages(table, ones, pools), lambda: ctx.compact_pages(table, pools)):
            with pytest.raises(psx.PsxError) as e:
                call()
            assert e.value.status == psx.ERR_BAD_ARGUMENT
    layout = psx.binding.PageTableLayout(table.pages.data_ptr(), table.lengths.data_ptr(), table.references.data_ptr(), 4, 4, 8, 16)
    lib, at = ctx._lib, C.addressof(layout)
    none = lambda **changed: [setattr(layout, k, v) for k, v in changed.items()]
    for changed, back in ((dict(pages=None), dict(pages=table.pages.data_ptr())), (dict(rows=-1), dict(rows=4)), (dict(max_pages=0), dict(max_pages=4)),
                          (dict(num_pages=0), dict(num_pages=8)), (dict(page_size=0), dict(page_size=16))):
        none(**changed)
        assert lib.psx_b200_extend_pages(ctx._ctx, None, at, ones.data_ptr(), None, 0, None) == psx.ERR_BAD_ARGUMENT
        assert lib.psx_b200_release_pages(ctx._ctx, None, at, None) == psx.ERR_BAD_ARGUMENT
        none(**back)
    assert lib.psx_b200_extend_pages(ctx._ctx, None, at, None, None, 0, None) == psx.ERR_BAD_ARGUMENT
    assert lib.psx_b200_extend_pages(ctx._ctx, None, at, ones.data_ptr(), None, 1, None) == psx.ERR_BAD_ARGUMENT
    assert lib.psx_b200_extend_pages(ctx._ctx, None, at, ones.data_ptr(), None, -1, None) == psx.ERR_BAD_ARGUMENT
    assert lib.psx_b200_fork_pages(ctx._ctx, None, at, ones.data_ptr(), 3) == psx.ERR_BAD_ARGUMENT
    assert lib.psx_b200_fork_pages(ctx._ctx, None, at, None, 2) == psx.ERR_BAD_ARGUMENT
    assert lib.psx_b200_compact_pages(ctx._ctx, None, at, None, 0, None) == psx.ERR_BAD_ARGUMENT
    for number, value in (("max_pages", 1 << 27), ("num_pages", (1 << 30) + 1)):
        none(**{number: value})
        assert lib.psx_b200_release_pages(ctx._ctx, None, at, None) == psx.ERR_UNSUPPORTED
        none(max_pages=4, num_pages=8)
    torch.cuda.synchronize()
    assert not table.lengths.any() and not table.references.any()
