"""kv_page_map_i32_cuda over many steps in which some requests are not served: whatever the steps,
no page is held twice, none is lost, and no token counts as stored that is not.

The model below knows lists and sets only; what the operator returns is held against the rules
of include/paged_ops.h and against these invariants, not against a restatement of its arithmetic.
"""

import ctypes
from ctypes import c_void_p

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev

I32 = np.int32


class Pool:
    """B request rows over a pool of pages, on the device, lengths and counters in place.
    held[b]: the pages that b really has; length[b]: its stored tokens; stuck[b]: the length that the
    device holds of a request that was not served and has not been set back, or None."""

    def __init__(self, B, P, width, num_pages, T, seed=0, ring=None):
        self.rng = np.random.default_rng(seed)
        self.B, self.P, self.width, self.num_pages, self.T = B, P, width, num_pages, T
        self.ring_size = ring or num_pages
        order = self.rng.permutation(num_pages).astype(I32)
        places = np.full(self.ring_size, -7, I32)
        places[:num_pages] = order[:self.ring_size]
        self.free = list(order)
        self.held, self.length, self.stuck = [[] for _ in range(B)], [0] * B, [None] * B
        self.table = dev(np.full((B, width), -1, I32))
        self.ring = dev(places)
        self.counters = dev(np.array([0, num_pages, 0], I32))
        self.lens, self.new = dev(np.zeros(B, I32)), dev(np.zeros(B, I32))
        self.start, self.pos, self.slots = (dev(np.full(k, 77, I32)) for k in (B + 1, T, T))

    def launch(self, stream=None):
        p = cf.KvPageMapParams(batch_size=self.B, num_tokens=self.T, page_size=self.P, num_pages=self.num_pages,
                               max_pages=self.width, ring_size=self.ring_size)
        return cf.call_op("kv_page_map_i32_cuda", [self.lens, self.new, self.counters],
                          [self.table, self.ring, self.lens, self.start, self.pos, self.slots, self.counters], p, stream)

    def set_back(self, b):
        """The caller's part of a second try: the length that the request really has."""
        lens = self.lens.download()
        lens[b] = self.length[b]
        self.lens.upload(lens)
        self.stuck[b] = None

    def step(self, new, run):
        """One step and everything that has to hold after it; the rows that were not served."""
        self.new.upload(np.asarray(new, I32))
        before = self.lens.download()
        run()
        lens, table, ring = self.lens.download(), self.table.download(), self.ring.download()
        head, avail, refused = (int(x) for x in self.counters.download())
        start, pos, slots = self.start.download(), self.pos.download(), self.slots.download()
        P, free, asked, row, missed, back = self.P, len(self.free), 0, 0, [], []
        taken = 0
        for b, n in enumerate(new):
            assert start[b] == row
            if n < 0:
                back += self.held[b]
                self.held[b], self.length[b], self.stuck[b] = [], 0, None
                assert lens[b] == 0
                continue
            mine = slots[row:row + n]
            assert self.stuck[b] is not None or (pos[row:row + n] == before[b] + np.arange(n)).all()
            row += n
            have, after = len(self.held[b]), -(-(self.length[b] + n) // P)
            if self.stuck[b] is not None:                 # its tokens of an earlier step are missing
                ok = False
            else:
                ok = after <= self.width
                if ok and after > have:
                    asked += after - have
                    ok = asked <= free
            if not ok:
                missed.append(b)
                assert (mine == -1).all()
                if self.stuck[b] is None:
                    self.stuck[b] = self.length[b] + n
                assert lens[b] == self.stuck[b]
                continue
            pages = [int(x) for x in table[b, :after]]
            assert pages[:have] == self.held[b]
            fresh = pages[have:]
            assert fresh == self.free[asked - len(fresh):asked], "pages in the ring's order"
            taken = asked if fresh else taken
            self.held[b], self.length[b] = pages, self.length[b] + n
            at = before[b] + np.arange(n)
            assert (mine == np.array(pages, I32)[at // P] * P + at % P).all()
            assert lens[b] == self.length[b]
        assert start[self.B] == row and (slots[row:] == -1).all() and (pos[row:] == -1).all()
        assert refused == len(missed)
        self.free = (self.free[taken:] + back)[:self.ring_size]
        assert avail == len(self.free)
        assert [int(ring[(head + j) % self.ring_size]) for j in range(avail)] == self.free
        everything = self.free + [p for h in self.held for p in h]
        assert len(set(everything)) == len(everything), "a page in two places"
        if self.ring_size >= self.num_pages:
            assert sorted(everything) == list(range(self.num_pages)), "a page lost"
        return missed


FORMS = [64, 5000]          # entries of positions and slots: one launch and two


def runner(gpu, pool, captured):
    st = cf.Stream()
    if not captured:
        def eager():
            assert pool.launch(st) == 0
            st.synchronize()
        return eager, lambda: None
    assert pool.launch(st) == 0                          # sizes the workspace; new_lens is 0
    st.synchronize()
    ex = c_void_p()
    assert gpu.gpu_capture_begin(st.handle) == 0
    assert pool.launch(st) == 0
    assert gpu.gpu_capture_end(st.handle, ctypes.byref(ex)) == 0

    def replay():
        assert gpu.gpu_graph_launch(ex, st.handle) == 0
        st.synchronize()
    return replay, lambda: gpu.gpu_graph_exec_destroy(ex)


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("T", FORMS)
def test_refused_then_ended(gpu, T, captured):
    """Four pages: A takes three, B finds too few, B ends, A ends; a request for all four then has
    them."""
    s = Pool(2, 16, 6, 4, T)
    run, end = runner(gpu, s, captured)
    assert s.step([40, 0], run) == []
    assert s.step([1, 20], run) == [1]
    assert s.step([0, -1], run) == []
    assert s.step([-1, 0], run) == []
    assert s.step([64, 0], run) == []
    end()


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("T", FORMS)
def test_refused_goes_on_unnoticed(gpu, T, captured):
    """A request whose token found no page decodes on: each step says that it is not served, until
    its length is set back and a page is free."""
    s = Pool(2, 16, 6, 3, T)
    run, end = runner(gpu, s, captured)
    assert s.step([32, 16], run) == []
    assert s.step([0, 1], run) == [1]
    for _ in range(3):
        assert s.step([0, 1], run) == [1]
    assert s.step([0, 0], run) == [1]                    # still without the tokens it was given
    assert s.step([-1, 1], run) == [1]
    s.set_back(1)
    assert s.step([0, 5], run) == []                     # fewer or more than it was refused
    assert s.step([0, 20], run) == []
    end()


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("T", FORMS)
def test_refused_past_the_table(gpu, T, captured):
    """A length past the table: not served, also with no new tokens, until it is set back; what it
    held before comes back when it ends."""
    s = Pool(3, 4, 3, 9, T)
    run, end = runner(gpu, s, captured)
    assert s.step([10, 12, 3], run) == []
    assert s.step([3, 1, 1], run) == [0, 1]
    assert s.step([0, 0, 1], run) == [0, 1]
    assert s.step([1, -1, 0], run) == [0]
    s.set_back(0)
    assert s.step([2, 12, 0], run) == []
    assert s.step([1, 1, 5], run) == [0, 1]
    assert s.step([-1, -1, -1], run) == []
    end()


@pytest.mark.gpu
@pytest.mark.parametrize("T", FORMS)
def test_ended_with_entries_that_are_no_pages(gpu, T):
    """A caller that has dropped the pages behind a window: the others come back, in their order."""
    P, width = 8, 200
    s = Pool(3, P, width, 400, T)
    run, end = runner(gpu, s, False)
    assert s.step([3, 0, 9], run) == []
    for n in (40, 62, 64, 40, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64):
        assert s.step([0, n, 0], run) == []
    table = s.table.download()
    have = len(s.held[1])
    assert have > 130
    dropped = [0, 1, 2, 63, 64, 100, 129]
    for j, what in zip(dropped, (-1, -1, -5, 400, -1, 2 ** 31 - 1, -2 ** 31)):
        table[1, j] = what
    s.table.upload(table)
    gone = [s.held[1][j] for j in dropped]
    s.held[1] = [p for j, p in enumerate(s.held[1]) if j not in dropped]
    s.held.append(gone)                                  # with the caller
    assert s.step([1, -1, -1], run) == []
    end()


@pytest.mark.gpu
@pytest.mark.parametrize("T", FORMS)
def test_ring_without_room_for_what_comes_back(gpu, T):
    """A ring of fewer places than pages: what comes back fills it; free pages in it stay."""
    s = Pool(4, 4, 8, 12, T, ring=16)
    run, end = runner(gpu, s, False)
    assert s.step([20, 12, 3, 0], run) == []             # 9 pages, 3 free in 16 places
    # The caller's own table rows name more pages than the ring was told of.
    s.held[3], s.length[3] = list(range(100, 108)), 32
    s.num_pages = 200
    lens, table = s.lens.download(), s.table.download()
    lens[3], table[3] = 32, np.arange(100, 108)
    s.lens.upload(lens), s.table.upload(table)
    assert s.ring_size < s.num_pages
    assert s.step([-1, -1, -1, -1], run) == []           # 17 for 13 places
    assert s.step([20, 1, 1, 1], run) == []
    end()


@pytest.mark.gpu
@pytest.mark.parametrize("T,B", [(64, 9), (5000, 9), (2000, 200), (20000, 1100), (30000, 2500)])
def test_many_steps_with_too_few_pages(gpu, T, B):
    """Random steps over a pool that is too small: requests retried with other lengths, left as
    they are, or ended, for a while."""
    P = 5
    s = Pool(B, P, 12, 3 * B, T, seed=B)
    run, end = runner(gpu, s, True)
    rng = np.random.default_rng(B + T)
    seen = 0
    for _ in range(40):
        new = rng.integers(0, 9, B)
        new[rng.random(B) < 0.35] = 0
        new[rng.random(B) < 0.12] = -1
        while np.maximum(new, 0).sum() > T:
            new[rng.random(B) < 0.5] = 0
        for b in range(B):
            if s.stuck[b] is not None and rng.random() < 0.5:
                s.set_back(b)
        seen += len(s.step([int(x) for x in new], run))
    assert seen > 10
    end()


@pytest.mark.gpu
@pytest.mark.parametrize("T", FORMS)
def test_a_row_of_almost_2_to_the_31_entries(gpu, T):
    """The longest row there can be, all of whose entries a request that is not served takes away
    (8 GiB): up to its end and not past it."""
    width, tail = 2 ** 31 - 1, 4096
    table = cf.DeviceBuffer(4 * (width + tail), I32)
    table.fill_zero()
    counters, ring, lens, new = (dev(np.array(x, I32)) for x in ([0, 3, 0], [5, 6, 7, 8], [1], [width]))
    start, pos, slots = (dev(np.full(k, 77, I32)) for k in (2, T, T))
    p = cf.KvPageMapParams(batch_size=1, num_tokens=T, page_size=1, num_pages=9, max_pages=width, ring_size=4)
    assert cf.call_op("kv_page_map_i32_cuda", [lens, new, counters], [table, ring, lens, start, pos, slots, counters], p) == 0
    assert list(counters.download()) == [0, 3, 1] and list(lens.download()) == [width]
    assert (slots.download() == -1).all() and (pos.download() == 1 + np.arange(T)).all()

    def entries(first, n):
        out = np.empty(n, I32)
        assert gpu.gpu_memcpy_d2h(out.ctypes.data, table.ptr + 4 * first, 4 * n, None) == 0
        return out
    assert entries(0, 1)[0] == 0
    for first in (1, 2 ** 30 - 2048, 2 ** 31 - 1 - 4096):
        assert (entries(first, 4096) == -1).all()
    assert (entries(width, tail) == 0).all()
    table.free()
