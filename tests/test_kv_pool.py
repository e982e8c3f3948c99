"""The pages of a K/V cache: fork, reserve, truncate, accept, compact and copy against a model that does one thing after the
other in numpy. Integers and copied rows have to be equal bit for bit."""
import numpy as np
import pytest

import lokal_b200 as L
from lokal_b200 import capi
from paged import PoolModel


# ---- no GPU ----

def test_null_arguments_are_refused():
    lib = capi.load()
    out = (capi.C.c_void_p * 1)()
    assert lib.lokal_cuda_kv_pool_create(None, 16, 1, 1, 1, None, None, None, None, 1, 16, out) == capi.ERR_BAD_ARG
    for name in ("reset", "compact", "destroy"):
        fn = getattr(lib, "lokal_cuda_kv_pool_" + name)
        assert fn(*[None] * len(fn.argtypes)) == capi.ERR_BAD_ARG
    for name in ("rows", "reserve", "fork", "truncate", "copy_pages", "accept"):
        fn = getattr(lib, "lokal_cuda_kv_pool_" + name)
        assert fn(*[0 if t in (capi.C.c_size_t, capi.C.c_uint32, capi.C.c_int64) else None for t in fn.argtypes]) == capi.ERR_BAD_ARG


def test_model_shares_copies_and_frees():
    m = PoolModel(8, 6, 3, 4, np.arange(2 * 48 * 1).reshape(2, 48, 1))
    m.reserve([0], [13])
    m.fork([0], [1])
    assert m.table[1, 0] == m.table[0, 0] == 0 and m.table[1, 1] == 2 and list(m.refs[:3]) == [2, 1, 1]
    assert (m.rows[:, 16:21] == m.rows[:, 8:13]).all()
    m.truncate([0])
    assert list(m.refs[:3]) == [1, 0, 1] and m.compact() == 2 and list(m.table[1, :2]) == [0, 1]
    m.reserve([2], [33])
    assert m.bad and not m.no_pages
    m.reserve([2, 0], [32, 8])
    assert not m.no_pages or m.lens[0] == 0


# ---- GPU ----

class Rig:
    """A pool on the device beside its model."""

    def __init__(self, ctx, dev, page, n_pages, n_slots, max_pages, n_stores, width, seed, shift=0):
        import torch
        self.torch, self.ctx = torch, ctx
        rng = np.random.default_rng(seed)
        rows = rng.integers(0, 65536, (n_stores, n_pages * page, width)).astype(np.uint16)
        self.m = PoolModel(page, n_pages, n_slots, max_pages, rows.copy())
        flat = torch.zeros(rows.size + 64, dtype=torch.int16, device="cuda")
        self.store = flat[shift:shift + rows.size].view(rows.shape)
        self.store.copy_(torch.from_numpy(rows.view(np.int16)))
        self.table = torch.full((n_slots, max_pages), 7, dtype=torch.int32, device="cuda")
        self.lens = torch.full((n_slots,), 7, dtype=torch.int32, device="cuda")
        self.refs = torch.full((n_pages,), 7, dtype=torch.int32, device="cuda")
        self.pool = L.KvPool(ctx, page_rows=page, n_pages=n_pages, n_slots=n_slots, max_pages=max_pages, table=self.table, lens=self.lens,
                             refs=self.refs, stores=[self.store[i] for i in range(n_stores)], row_bytes=2 * width)
        self.pool.reset()

    def ints(self, a):
        return self.torch.tensor(np.asarray(a, np.int64).astype(np.uint32).view(np.int32), device="cuda") if len(a) else \
            self.torch.zeros(1, dtype=self.torch.int32, device="cuda")

    def sync(self):
        try:
            self.ctx.stream_sync()
            return capi.OK
        except L.LokalCudaError as e:
            return e.status

    def same(self, what):
        status = self.sync()
        want = capi.ERR_NO_PAGES if self.m.no_pages else capi.ERR_PAGE_RANGE if self.m.bad else capi.OK
        assert status == want, what
        self.m.no_pages = self.m.bad = False
        assert np.array_equal(self.lens.cpu().numpy(), self.m.lens), what
        assert np.array_equal(self.table.cpu().numpy(), self.m.table), what
        assert np.array_equal(self.refs.cpu().numpy(), self.m.refs), what
        assert np.array_equal(self.store.cpu().numpy().view(np.uint16), self.m.rows), what
        held = np.bincount(self.m.table[self.m.table >= 0], minlength=self.m.n_pages)
        assert np.array_equal(held, self.m.refs), what

    def both(self, name, *lists):
        getattr(self.m, name)(*lists)
        getattr(self.pool, name)(*[None if a is None else self.ints(a) for a in lists], n=len(lists[0]))

    def accept(self, slots, n_rows, accepted, counts):
        self.m.accept(slots, n_rows, accepted, counts)
        starts = np.concatenate([[0], np.cumsum(n_rows)])
        self.pool.accept(self.ints(slots), self.ints(starts), self.ints(np.asarray(accepted).reshape(-1)), self.ints(counts), n_seqs=len(slots),
                         max_accept=np.asarray(accepted).shape[1])


@pytest.mark.gpu
@pytest.mark.parametrize("page,n_pages,n_slots,max_pages,n_stores,width,shift", [
    (8, 40, 9, 10, 4, 8, 0), (16, 300, 40, 12, 6, 72, 0), (64, 24, 7, 5, 2, 512, 0), (256, 9, 5, 3, 2, 24, 0),
    (16, 60, 12, 9, 3, 5, 0),      # rows of ten bytes: no 16-byte accesses
    (16, 60, 12, 9, 3, 16, 1),     # stores that are only 2-byte aligned
    (8, 5000, 30, 400, 2, 8, 0),   # more pages than one pass of the plan's scan takes
])
def test_any_order_of_calls_matches_the_model(ctx, dev, page, n_pages, n_slots, max_pages, n_stores, width, shift):
    r = Rig(ctx, dev, page, n_pages, n_slots, max_pages, n_stores, width, page + n_pages, shift)
    rng = np.random.default_rng(n_pages)
    r.same("empty")
    cap = page * max_pages
    for step in range(40):
        name = rng.choice(["reserve", "reserve", "fork", "truncate", "accept", "compact"])
        k = int(rng.integers(1, n_slots + 1))
        slots = rng.permutation(n_slots)[:k]
        if name == "reserve":
            r.both("reserve", slots, np.minimum(cap, r.m.lens[slots] + rng.integers(0, 4 * page, k)))
        elif name == "fork":
            empty = np.flatnonzero(r.m.lens == 0)[:k]
            if len(empty):
                r.both("fork", rng.integers(0, n_slots, len(empty)), empty)
        elif name == "truncate":
            k = max(1, k // 3)
            if rng.random() < 0.3:
                r.both("truncate", slots[:k], None)
            else:
                r.both("truncate", slots[:k], (r.m.lens[slots[:k]] * rng.random(k)).astype(int))
        elif name == "accept":
            # rows may be moved only in pages that no other slot holds: grow first, as a program does before it drafts
            drafts = rng.integers(0, 12, k)
            want = np.minimum(cap, r.m.lens[slots] + drafts)
            r.both("reserve", slots, want)
            ok = r.m.lens[slots] == want
            n = np.where(ok, drafts, 0)
            n = np.minimum(n, r.m.lens[slots])
            counts = np.array([rng.integers(0, x + 1) for x in n])
            acc = np.zeros((k, 12), np.int64)
            for i in range(k):
                acc[i, :counts[i]] = np.sort(rng.permutation(n[i])[:counts[i]])
            r.accept(slots, n, acc, counts)
        else:
            used = r.torch.zeros(1, dtype=r.torch.int32, device="cuda")
            r.pool.compact(used)
            assert r.m.compact() == int(used.item())
        r.same(f"step {step}: {name}")


@pytest.mark.gpu
def test_accept_moves_rows_in_place_when_targets_are_later_sources(ctx, dev):
    # the path 1, 2, 3, ... moves to 0, 1, 2, ...: every target is the next move's source; 31 moves cross pages and batches
    for page in (8, 16):
        r = Rig(ctx, dev, page, 12, 2, 8, 3, 40, page)
        r.both("reserve", [1], [5 + 32])
        r.accept([1], [32], [list(range(1, 32))], [31])
        r.same("a chain shifted by one")
        assert r.m.lens[1] == 36
        r.accept([1], [4], [[0, 2]], [2])
        r.same("the first stays")
        r.accept([1], [3], [[0, 0]], [0])
        r.same("none accepted")


@pytest.mark.gpu
def test_writers_of_a_shared_partly_filled_page_get_their_own(ctx, dev):
    # a fork cut back into a page that its source still holds: whoever grows first takes a copy
    r = Rig(ctx, dev, 16, 20, 4, 6, 2, 64, 3)
    r.both("reserve", [0], [48])
    r.both("fork", [0, 0], [1, 2])
    r.both("truncate", [1, 2], [37, 41])
    r.same("shared last page")
    assert r.m.refs[r.m.table[0, 2]] == 3
    r.both("reserve", [1, 2, 0], [40, 60, 48])
    r.same("copied before it is written")
    assert r.m.refs[r.m.table[0, 2]] == 1 and len({int(r.m.table[i, 2]) for i in range(3)}) == 3


@pytest.mark.gpu
def test_pages_run_out_in_list_order(ctx, dev):
    r = Rig(ctx, dev, 8, 10, 6, 8, 2, 8, 5)
    r.both("reserve", [0, 1, 2, 3, 4], [24, 40, 32, 8, 0])  # 3 + 5 fit, 4 do not, and the one after it is not served either
    assert r.m.no_pages and list(r.m.lens[:5]) == [24, 40, 0, 0, 0]
    r.same("exhausted")
    r.both("truncate", [1, 1, 0], [17, 9, 50])  # the smaller of the two lengths of slot 1
    r.same("given back")
    assert r.m.lens[1] == 9 and r.m.lens[0] == 24
    r.both("fork", [1, 1, 1, 1, 1, 1], [2, 3, 4, 5, 2, 9])  # slot 2 twice, and one that is not there
    assert r.m.bad
    r.same("forks")
    r.both("truncate", [0, 1, 2, 3, 4, 5], None)
    r.same("all freed")
    assert not r.m.refs.any()


@pytest.mark.gpu
def test_bad_entries_change_nothing_and_are_reported(ctx, dev):
    r = Rig(ctx, dev, 8, 12, 4, 4, 2, 8, 7)
    r.both("reserve", [0, 1], [12, 20])
    r.same("start")
    for name, lists in [("reserve", ([9], [8])), ("reserve", ([0], [33])), ("reserve", ([0], [-1])), ("reserve", ([2, 2], [8, 16])),
                        ("fork", ([0], [1])), ("fork", ([0], [0])), ("fork", ([7], [2])), ("truncate", ([4], [0])), ("truncate", ([0], [-5]))]:
        r.both(name, *lists)
        assert r.m.bad, (name, lists)
        r.same(f"{name} {lists}")
    for n, acc, count in [([4], [[2, 1]], [2]), ([4], [[1, 1]], [2]), ([4], [[0, 4]], [2]), ([4], [[-1, 2]], [2]), ([4], [[0, 1]], [5]),
                          ([30], [[0, 1]], [2]), ([4], [[0, 1]], [-1])]:
        r.accept([1], n, acc, count)
        assert r.m.bad
        r.same(f"accept {n} {acc} {count}")
    r.accept([1, 1], [2, 2], [[1], [1]], [1, 1])
    assert r.m.bad
    r.same("one slot twice")


@pytest.mark.gpu
def test_pages_are_copied_and_rows_are_found(ctx, dev):
    import torch
    r = Rig(ctx, dev, 16, 40, 4, 6, 3, 24, 11)
    src, dst = [0, 5, 39, 5], [10, 11, 12, 13]
    r.pool.copy_pages(r.ints(src), r.ints(dst), n=4)
    for a, b in zip(src, dst):
        r.m._copy(a, b, 16)
    r.same("copied")
    r.pool.copy_pages(r.ints([0, 40]), r.ints([-1, 3]), n=2)
    r.m.bad = True
    r.same("pages that are not there")
    r.both("reserve", [3, 1], [50, 17])
    r.same("reserved")
    pos = np.array([0, 15, 16, 49, 50, -1, 16, 17, 3], np.int32)
    slots = np.array([3, 3, 3, 3, 3, 1, 1, 1, 8], np.uint32)
    out = torch.zeros(9, dtype=torch.int32, device="cuda")
    r.pool.rows(out, rows=9, positions=r.ints(pos), slots=r.ints(slots))
    assert r.sync() == capi.ERR_POS_RANGE
    want = [r.m.row(s, p) if s < 4 and 0 <= p < r.m.lens[s] else capi.KV_ROW_NONE for s, p in zip(slots, pos)]
    assert np.array_equal(out.cpu().numpy().view(np.uint32), np.array(want, np.uint32))
    r.pool.rows(out, rows=9, pos0=9, slot0=3)
    assert r.sync() == capi.OK
    assert list(out.cpu().numpy()) == [r.m.row(3, 9 + i) for i in range(9)]


@pytest.mark.gpu
def test_a_captured_step_replays_on_the_state_it_finds(ctx, dev):
    r = Rig(ctx, dev, 8, 64, 8, 12, 2, 16, 13)
    r.both("reserve", [0, 1], [13, 30])
    r.same("start")
    src, dst, grow, want, none = r.ints([0, 1]), r.ints([2, 3]), r.ints([2, 3]), r.ints([40, 41]), r.ints([0, 1])
    s = ctx.stream_create()
    ctx.graph_begin(s)
    r.pool.fork(src, dst, n=2, stream=s)
    r.pool.reserve(grow, want, n=2, stream=s)
    r.pool.compact(stream=s)
    graph = ctx.graph_end(s)
    r.same("capturing changes nothing")
    for cut in ([13, 30], [8, 17], [0, 1]):
        ctx.graph_launch(graph, s)
        ctx.stream_sync(s)
        r.m.fork([0, 1], [2, 3])
        r.m.reserve([2, 3], [40, 41])
        r.m.compact()
        r.same(f"replayed {cut}")
        r.both("truncate", [2, 3], None)
        r.both("truncate", [0, 1], cut)
        r.same(f"cut {cut}")
    ctx.graph_destroy(graph)
    ctx.stream_destroy(s)


@pytest.mark.gpu
def test_create_refusals(ctx, dev):
    import torch
    t = torch.zeros(4096, dtype=torch.int32, device="cuda")
    good = dict(page_rows=16, n_pages=4, n_slots=2, max_pages=2, table=t, lens=t[64:], refs=t[128:], stores=[t[256:]], row_bytes=16)
    L.KvPool(ctx, **good).close()
    for bad, status in [(dict(page_rows=4), capi.ERR_BAD_ARG), (dict(page_rows=24), capi.ERR_BAD_ARG), (dict(page_rows=512), capi.ERR_BAD_ARG),
                        (dict(n_pages=0), capi.ERR_BAD_ARG), (dict(n_slots=0), capi.ERR_BAD_ARG), (dict(max_pages=0), capi.ERR_BAD_ARG),
                        (dict(stores=[]), capi.ERR_BAD_ARG), (dict(row_bytes=0), capi.ERR_BAD_ARG), (dict(row_bytes=7), capi.ERR_BAD_ARG),
                        (dict(n_pages=1 << 27), capi.ERR_BAD_ARG), (dict(max_pages=1 << 28), capi.ERR_BAD_ARG), (dict(table=None), capi.ERR_BAD_ARG),
                        (dict(stores=[None]), capi.ERR_BAD_ARG), (dict(lens=t.data_ptr() + 2), capi.ERR_MISALIGNED),
                        (dict(stores=[t.data_ptr() + 1]), capi.ERR_MISALIGNED)]:
        with pytest.raises(L.LokalCudaError) as e:
            L.KvPool(ctx, **{**good, **bad})
        assert e.value.status == status, bad
    pool = L.KvPool(ctx, **good)
    for call in (lambda: pool.reserve(t, t, n=3), lambda: pool.reserve(t, None, n=1), lambda: pool.fork(None, t, n=1),
                 lambda: pool.copy_pages(t, t, n=5), lambda: pool.accept(t, t, t, t, n_seqs=1, max_accept=257),
                 lambda: pool.accept(t, t, None, t, n_seqs=1, max_accept=1), lambda: pool.rows(None, rows=1), lambda: pool.rows(t, rows=1, pos0=-1)):
        with pytest.raises(L.LokalCudaError) as e:
            call()
        assert e.value.status == capi.ERR_BAD_ARG
    with pytest.raises(L.LokalCudaError) as e:
        pool.truncate(t.data_ptr() + 1, n=1)
    assert e.value.status == capi.ERR_MISALIGNED
    pool.reserve(None, None, n=0)
    pool.fork(None, None, n=0)
    ctx.stream_sync()
    pool.close()


@pytest.mark.gpu
def test_the_longest_slot_leaves_room_for_a_tile(ctx, dev):
    import torch
    t = torch.zeros(4096, dtype=torch.int32, device="cuda")
    good = dict(page_rows=16, n_pages=4, n_slots=2, table=t, lens=t[64:], refs=t[128:], stores=[t[256:]], row_bytes=16)
    most = (2 ** 31 - 256) // 16
    L.KvPool(ctx, max_pages=most, **good).close()
    with pytest.raises(L.LokalCudaError) as e:
        L.KvPool(ctx, max_pages=most + 1, **good)
    assert e.value.status == capi.ERR_BAD_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("page,n_stores,width", [(16, 6, 512), (8, 2, 5)])
def test_a_slot_that_accept_names_many_times_belongs_to_the_first(ctx, dev, page, n_stores, width):
    """The later entries find the slot while the first one cuts it: behind the cut its length is shorter than their drafts."""
    r = Rig(ctx, dev, page, 600, 48, 24, n_stores, width, 23)
    rng = np.random.default_rng(23)
    for step in range(25):
        slots = rng.integers(0, 6, 48)
        grow = rng.integers(20, 60, 6)
        r.both("reserve", np.arange(6), r.m.lens[:6] + grow)
        n = grow[slots]
        counts = np.array([int(rng.integers(0, 9)) for _ in slots])
        acc = np.stack([np.sort(rng.permutation(k)[:8]) for k in n])
        r.accept(slots, n, acc, counts)
        r.same(f"step {step}")
        r.both("truncate", np.arange(6), rng.integers(0, 30, 6))
        r.same(f"cut {step}")


@pytest.mark.gpu
def test_a_new_pool_is_ready_on_any_stream(ctx, dev):
    """The first call on a pool is a fork on a stream that does not order itself behind the default one: it reads the addresses
    of the stores that create has sent to the device."""
    import torch
    page, n_stores = 8, 300
    s = ctx.stream_create()
    for step in range(40):
        store = torch.full((n_stores, 8 * page, 8), step, dtype=torch.int16, device="cuda")
        store[:, 2 * page:] = -1
        table = torch.tensor([[0, 1], [-1, -1]], dtype=torch.int32, device="cuda")
        lens = torch.tensor([13, 0], dtype=torch.int32, device="cuda")
        refs = torch.tensor([1, 1, 0, 0, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
        src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 1))
        torch.cuda.synchronize()
        pool = L.KvPool(ctx, page_rows=page, n_pages=8, n_slots=2, max_pages=2, table=table, lens=lens, refs=refs,
                        stores=[store[i] for i in range(n_stores)], row_bytes=16)
        pool.fork(src, dst, n=1, stream=s)
        ctx.stream_sync(s)
        assert table[1].tolist() == [0, 2] and refs.tolist()[:3] == [2, 1, 1]
        assert (store[:, 2 * page:2 * page + 5] == step).all() and (store[:, 2 * page + 5:] == -1).all()
        pool.close()
    ctx.stream_destroy(s)


class CarefulModel(PoolModel):
    """accept leaves a sequence as it was if a row would move into a page that another slot holds before the call."""

    def accept(self, slots, n_rows, accepted, counts):
        refs, seen, counts = self.refs.copy(), set(), list(counts)
        for i, (s, n) in enumerate(zip(slots, n_rows)):
            if s in seen or s >= self.n_slots:
                continue
            seen.add(s)
            base = int(self.lens[s]) - n
            moves = [base + j for j, a in enumerate(list(accepted[i])[:max(0, counts[i])]) if a != j and 0 <= base + j < self.max_pages * self.page]
            if any(refs[self.table[s, p // self.page]] > 1 for p in moves if self.table[s, p // self.page] >= 0):
                counts[i] = -1
        super().accept(slots, n_rows, accepted, counts)


@pytest.mark.gpu
def test_accept_does_not_move_rows_into_a_page_that_another_slot_holds(ctx, dev):
    r = Rig(ctx, dev, 8, 40, 6, 8, 3, 40, 29)
    r.m.__class__ = CarefulModel
    r.both("reserve", [0], [8 + 16])  # 8 committed rows, two pages of drafted ones
    r.both("fork", [0, 0], [1, 2])
    r.same("forked between drafting and accepting")
    r.accept([0], [16], [[1, 2]], [2])
    assert r.m.bad and r.m.lens[0] == 24
    r.same("shared target")
    r.accept([0, 1], [16, 16], [[0, 1], [0, 9]], [2, 2])  # no row of 0 moves, so it is cut; one of 1 does, and would into a shared page
    assert r.m.bad and r.m.lens[0] == 10 and r.m.lens[1] == 24
    r.same("only what moves counts")
    r.accept([1, 2], [16, 16], [[0, 0], [5, 8]], [0, 2])  # 1 gives its pages back in the call in which 2 would write into one of them
    assert r.m.bad and r.m.lens[1] == 8 and r.m.lens[2] == 24
    r.same("the counts are those of before the call")
    r.accept([2], [8], [[3, 7]], [2])  # the last page is its own by now
    assert not r.m.bad and r.m.lens[2] == 18
    r.same("its own page")


@pytest.mark.gpu
@pytest.mark.parametrize("page,n_slots,n_stores,width", [(8, 12, 40, 512), (16, 70, 3, 24), (16, 300, 2, 8)])
def test_accept_on_slots_that_share_pages_in_any_order(ctx, dev, page, n_slots, n_stores, width):
    r = Rig(ctx, dev, page, 40 * n_slots // 8, n_slots, 10, n_stores, width, 31)
    r.m.__class__ = CarefulModel
    rng = np.random.default_rng(31)
    refused = 0
    for step in range(12):
        roots = n_slots // 4
        r.both("truncate", np.arange(n_slots), None)
        r.both("reserve", np.arange(roots), rng.integers(page, 5 * page, roots))
        r.both("fork", rng.integers(0, roots, n_slots - roots), np.arange(roots, n_slots))
        some = rng.permutation(n_slots)[:n_slots // 3]
        r.both("reserve", some, np.minimum(10 * page, r.m.lens[some] + rng.integers(1, 2 * page, len(some))))
        r.same(f"step {step}: made")
        slots = rng.permutation(n_slots)
        n = np.array([int(rng.integers(0, r.m.lens[s] + 1)) for s in slots])
        counts = np.array([int(rng.integers(0, min(x, 12) + 1)) for x in n])
        acc = np.zeros((n_slots, 12), np.int64)
        for i in range(n_slots):
            acc[i, :counts[i]] = np.arange(counts[i]) if rng.random() < 0.3 else np.sort(rng.permutation(n[i])[:counts[i]])
        r.accept(slots, n, acc, counts)
        refused += r.m.bad
        r.same(f"step {step}: accepted")
    assert refused


@pytest.mark.gpu
def test_a_step_that_runs_out_of_pages_says_so(ctx, dev):
    """What follows in the step finds the rows missing too; the status is the one that a scheduler acts on."""
    import torch
    r = Rig(ctx, dev, 8, 4, 3, 4, 2, 8, 37)
    out = torch.zeros(24, dtype=torch.int32, device="cuda")
    r.both("reserve", [0, 1], [16, 24])
    r.pool.rows(out, rows=24, slot0=1)
    ctx.tree_plan(r.pool, slots=r.ints([1]), q_start=r.ints([0, 24]), n_seqs=1, rows=24, cache_rows=out)
    assert r.m.no_pages
    r.same("reserve, rows and plan of a step")
    r.pool.rows(out, rows=24, slot0=1)
    assert r.sync() == capi.ERR_POS_RANGE


@pytest.mark.gpu
def test_a_host_pass_reports_what_a_pool_call_before_it_met(ctx, dev):
    """run_host returns with the errors of the context, whichever call met them."""
    import torch
    from synth import BF16
    from test_gpu_pass import build_pass, inputs_on, make_case, pass_inputs
    cfg, a = make_case(BF16)
    p = build_pass(ctx, dev, cfg, a, slots=2)
    th = inputs_on("host", dev, cfg, a)
    out = torch.zeros(cfg.rows, cfg.hidden, dtype=dev.tdt[BF16]).pin_memory()
    r = Rig(ctx, dev, 8, 4, 3, 4, 2, 8, 39)
    for slots, lens, status in [([0], [33], capi.ERR_PAGE_RANGE), ([0, 1], [16, 24], capi.ERR_NO_PAGES)]:
        r.pool.reserve(r.ints(slots), r.ints(lens), n=len(slots))
        torch.cuda.synchronize()
        with pytest.raises(L.LokalCudaError) as e:
            p.run_host(pass_inputs(cfg, th, 7), out)
        assert e.value.status == status
        p.run_host(pass_inputs(cfg, th, 7), out)
    p.close()


class FakeLib:
    """Stands in for the library: hands out a handle and remembers what is destroyed."""

    def __init__(self):
        self.gone = []

    def lokal_cuda_create(self, device, out):
        out._obj.value = 7
        return capi.OK

    def lokal_cuda_kv_pool_create(self, *args):
        args[-1]._obj.value = 0x1234
        return capi.OK

    def lokal_cuda_kv_pool_destroy(self, ctx, pool):
        self.gone.append(("pool", ctx.value, pool.value))
        return capi.OK

    def lokal_cuda_destroy(self, ctx):
        self.gone.append(("context", ctx.value))


def test_a_context_that_is_closed_first_takes_its_pools_along(monkeypatch):
    monkeypatch.setattr(capi, "load", FakeLib)
    ctx = L.Context(0)
    made = [L.KvPool(ctx, page_rows=16, n_pages=1, n_slots=1, max_pages=1, table=1, lens=1, refs=1, stores=[1], row_bytes=16) for _ in range(2)]
    made[0].close()
    ctx.close()
    made[1].close()
    ctx.close()
    assert ctx._lib.gone == [("pool", 7, 0x1234), ("pool", 7, 0x1234), ("context", 7)]
