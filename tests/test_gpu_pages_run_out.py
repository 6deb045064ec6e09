"""A cache in pages whose pool runs out while rows share pages (psx_b200_extend_pages with psx_b200_rotate_heads): whatever rows are served, and
whatever they then store, every row goes on seeing the positions that it holds.  Numbers are stored as they come, without norm or rotation, so everything is
equal."""
import numpy as np
import pytest

import gpu_harness as gh
import pulsatrix_b200 as psx
import test_gpu_page_table as table_test

pytestmark = pytest.mark.gpu
HEADS, DIM = 2, 8


def _whole(values, kind="int64"):
    import torch
    return torch.tensor(values, dtype=getattr(torch, kind), device="cuda")


class _Rows:
    """A table with one layer, and beside it what every row holds: a number of its own for every position, kept row by row without any page."""

    def __init__(self, rows, max_pages, num_pages, size):
        import torch
        self.table = psx.PageTable.empty(rows, max_pages, num_pages, size)
        self.cache = psx.PagedCache(self.table, *[torch.full((num_pages, HEADS, size, DIM), -1.0, device="cuda") for _ in range(2)])
        self.held = [np.zeros(0, np.float32) for _ in range(rows)]
        self.stored = 0

    def extend(self, added):
        """Room, and new positions for the rows that get it; the others ask too, and store nothing."""
        import torch
        ctx, rows = gh.ctx(), len(self.held)
        first = self.table.lengths.clone()
        status = ctx.extend_pages(self.table, _whole(added), self.cache.pools()).tolist()
        counts = [max(0, n) for n in added]
        offsets = np.concatenate([[0], np.cumsum(counts)])
        new = (self.stored + np.arange(offsets[-1])).astype(np.float32)
        self.stored += len(new)
        x = torch.from_numpy(new).cuda()[:, None, None].expand(-1, HEADS, DIM).contiguous()
        _, _, kept = ctx.rotate_heads(x, x, -x, offsets=_whole(offsets.tolist()), first=first, cache=self.cache)
        for b, n in enumerate(counts):
            assert (kept[b] == psx.ROW_OK) == (status[b] == psx.ROW_OK or n == 0)
            if status[b] == psx.ROW_OK:
                self.held[b] = np.concatenate([self.held[b], new[offsets[b]:offsets[b + 1]]])
        return status

    def fork(self, parents):
        gh.ctx().fork_pages(self.table, _whole(parents))
        beams = len(parents[0])
        self.held = [self.held[b // beams * beams + p] for b, p in enumerate(np.asarray(parents).reshape(-1))]

    def release(self, keep):
        gh.ctx().release_pages(self.table, _whole(keep))
        self.held = [x[:max(n, 0)] for x, n in zip(self.held, keep)]

    def check(self):
        table, size = self.table.pages.cpu().numpy(), self.table.page_size
        assert self.table.lengths.tolist() == [len(x) for x in self.held]
        used, pools = np.zeros(self.table.num_pages, np.int32), [p.cpu().numpy() for p in self.cache.pools()]
        for b, x in enumerate(self.held):
            position = np.arange(len(x))
            at = table[b][position // size], slice(None), position % size
            assert (pools[0][at] == x[:, None, None]).all() and (pools[1][at] == -x[:, None, None]).all(), b
            np.add.at(used, table[b][:-(-len(x) // size)], 1)
        assert self.table.references.tolist() == used.tolist()


@pytest.mark.parametrize("size", [16, 64])
@pytest.mark.parametrize("keep,free,status", [((5, 4), 0, (64, 64)), ((4, 5), 0, (64, 0)), ((5, 5), 0, (64, 0)), ((5, 4), 1, (0, 0)),
                                              ((3, 9, 6), 1, (0, 64, 64)), ((9, 3, 6), 1, (0, 64, 0)), ((9, 3, 6), 0, (64, 64, 64)), ((2, 3, 6), 0, (64, 64, 0)),
                                              ((7, 3, 6, 1), 2, (0, 0, 64, 64)), ((7, 3, 6, 1), 3, (0, 0, 0, 0))])
def test_rows_that_go_on_in_one_page_with_different_numbers_of_positions(size, keep, free, status):
    # a page is kept in place by the last row that goes on in it, but never over what a row holds that got no page
    rows = _Rows(len(keep), 2, 1 + free, size)
    rows.extend([12] + [0] * (len(keep) - 1))
    rows.fork([[0] * len(keep)])
    rows.release(list(keep))
    rows.check()
    before = rows.table.pages.tolist(), rows.table.lengths.tolist()
    assert rows.extend([1] * len(keep)) == list(status)
    rows.check()
    for b, refused in enumerate(status):
        assert not refused or (rows.table.pages[b].tolist()[:1] == before[0][b][:1] and int(rows.table.lengths[b]) == before[1][b])
    # with pages given back the refused ones go on
    if any(status):
        last = len(keep) - 1
        rows.release([keep[0] + 1] + [0] * last)
        rows.check()
        assert rows.extend([1] * len(keep))[0] == 0
        rows.check()


def test_a_kept_page_and_more_pages_beside_it():
    # the last row asks for whole pages, too, which are not there; the row before it holds less than it, and more
    for keep in ((5, 9), (9, 5)):
        rows = _Rows(2, 4, 2, 16)
        rows.extend([12, 0])
        rows.fork([[0, 0]])
        rows.release(list(keep))
        assert rows.extend([1, 20]) == [0, 64]
        rows.check()
        rows = _Rows(3, 4, 2, 16)
        rows.extend([12, 0, 16])
        rows.fork([[0, 0, 2]])
        rows.release([*keep, 16])
        assert rows.extend([1, 1, 0]) == [64, 0 if keep[1] >= keep[0] else 64, 0]
        rows.check()


@pytest.mark.parametrize("groups,beams,num_pages,seed", [(1, 2, 3, 0), (2, 3, 8, 1), (7, 5, 30, 2), (3, 8, 20, 3), (1, 64, 60, 4), (40, 30, 300, 5)])
def test_every_row_sees_what_it_holds(groups, beams, num_pages, seed):
    rng = np.random.RandomState(seed)
    rows, size, max_pages = groups * beams, 16, 5
    run = _Rows(rows, max_pages, num_pages, size)
    for step in range(60):
        call = rng.randint(0, 10) if step > 1 else 0
        if call < 5:
            run.extend((rng.randint(0, rng.choice([2, 5, 30]), rows) * (rng.rand(rows) < 0.9)).tolist())
        elif call < 7:
            run.fork(rng.randint(0, beams, (groups, beams)).tolist())
        elif call < 9:
            run.release([int(len(x) * rng.choice([0, 0.5, 0.8, 0.95, 1], p=[0.1, 0.1, 0.2, 0.3, 0.3])) for x in run.held])
        else:
            gh.ctx().compact_pages(run.table, run.cache.pools())
        run.check()


class _Book(table_test.Book):
    """The restatement of test_gpu_page_table.py, in which a row that keeps its page is refused, too, where it would write over a refused row's positions."""

    def extend(self, added):
        size = self.size
        before, held, most = list(self.lengths), list(self.references), self.most * size
        going = {}
        for b, n in enumerate(added):
            if n > 0 and before[b] + n <= most and before[b] % size:
                going.setdefault(self.table[b][before[b] // size], []).append(b)
        entry = {b: self.table[b][before[b] // size] for rows in going.values() for b in rows}
        status = super().extend(added)
        for page, rows in going.items():
            keeper = rows[-1]
            over = [b for b in rows[:-1] if status[b] == psx.ROW_CACHE_FULL and before[b] % size > before[keeper] % size]
            if held[page] > 1 and len(rows) == held[page] and over and status[keeper] == 0:
                assert -(-before[keeper] // size) == -(-(before[keeper] + added[keeper]) // size) and entry[keeper] == page  # (it asked for no page)
                self.lengths[keeper], status[keeper] = before[keeper], psx.ROW_CACHE_FULL
        return status


@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("groups,beams,num_pages,seed", [(7, 5, 30, 4), (7, 5, 30, 6), (7, 5, 40, 7), (1, 64, 100, 8), (2, 3, 7, 9)])
def test_a_run_of_calls_where_pages_run_out(size, groups, beams, num_pages, seed, monkeypatch):
    monkeypatch.setattr(table_test, "Book", _Book)
    table_test.test_a_run_of_calls(size, groups, beams, num_pages, seed)
