"""Attention of drafted rows over a paged cache, and the plan that makes its masks, against a plain f64 form on the CPU.
Tolerances are the bound of tests/paged.py::tolerance, element for element."""
import numpy as np
import pytest

import lokal_b200 as L
import synth
from lokal_b200 import capi
from paged import attention, tolerance, visible
from synth import BF16, F16, F32


def test_null_arguments_are_refused():
    lib = capi.load()
    for name in ("lokal_cuda_tree_plan", "lokal_cuda_tree_attn"):
        fn = getattr(lib, name)
        assert fn(*[None if t is capi.C.c_void_p else 0 for t in fn.argtypes]) == capi.ERR_BAD_ARG
    assert lib.lokal_cuda_tree_attn_workspace(None, 1, 1, 1, 64) == 0


def random_parents(rng, n):
    return np.array([int(rng.integers(max(-1, j - 6), j)) for j in range(n)], np.int32)


def mask_of(parents, words):
    out = np.zeros((len(parents), words), np.uint64)
    for j, p in enumerate(parents):
        if p >= 0:
            out[j] = out[p]
        out[j, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


def bits(rows, words, rng):
    return rng.integers(0, 2 ** 63, (rows, words)).astype(np.uint64) * np.uint64(2) + rng.integers(0, 2, (rows, words)).astype(np.uint64)


class Case:
    """Sequences of a pool, their rows and the cache, on both sides."""

    def __init__(self, ctx, dev, *, lens, drafts, hq, hkv, hd, page=16, dtype=F32, kv=F32, mask="tree", seed=0, pad=0, q_pad=0, scale=None,
                 k_scale=1.0, extra_rows=0, slots=None, spare=2):
        import torch
        self.torch, self.ctx, self.dev = torch, ctx, dev
        rng = np.random.default_rng(seed)
        self.lens, self.drafts = np.asarray(lens, np.int64), np.asarray(drafts, np.int64)
        self.hq, self.hkv, self.hd, self.page, self.dtype, self.kv = hq, hkv, hd, page, dtype, kv
        self.scale = hd ** -0.5 if scale is None else scale
        n = len(lens)
        self.slots = np.arange(n) if slots is None else np.asarray(slots)
        held = -(-self.lens // page)
        self.n_pages = int(held.sum()) + spare
        self.max_pages = int(held.max()) + 1
        self.n_slots = int(self.slots.max()) + 2
        order = rng.permutation(self.n_pages)
        self.table = np.full((self.n_slots, self.max_pages), -1, np.int32)
        at = 0
        for i in range(n):
            self.table[self.slots[i], :held[i]] = order[at:at + held[i]]
            at += held[i]
        self.starts = np.concatenate([[0], np.cumsum(self.drafts)])
        self.rows = int(self.starts[-1]) + extra_rows
        self.width = hkv * hd + pad
        self.k = synth.round_to(rng.standard_normal((self.n_pages * page, self.width), dtype=np.float32) * np.float32(k_scale), kv)
        self.v = synth.round_to(rng.standard_normal((self.n_pages * page, self.width), dtype=np.float32), kv)
        self.q = synth.round_to(rng.standard_normal((self.rows, hq * hd + q_pad), dtype=np.float32), dtype)
        words = max(1, -(-int(self.drafts.max()) // 64))
        self.mask = None
        if mask == "tree":
            self.mask = np.concatenate([mask_of(random_parents(rng, int(d)), words) for d in self.drafts] + [np.zeros((extra_rows, words), np.uint64)])
        elif mask == "random":
            self.mask = bits(self.rows, words, rng)
        elif mask == "none":
            self.mask = np.zeros((self.rows, words), np.uint64)
        self.words = words
        self.fill = 7.0

    def cache_row(self, i, pos):
        return self.table[self.slots[i], pos // self.page].astype(np.int64) * self.page + pos % self.page

    def upload(self):
        put, t = self.dev.put, self.torch
        d = {"table": put(self.table), "k": put(self.k, self.kv), "v": put(self.v, self.kv), "q": put(self.q, self.dtype)}
        lens = np.zeros(self.n_slots, np.int32)
        lens[self.slots] = self.lens
        d["lens"] = put(lens)
        d["refs"] = t.zeros(self.n_pages, dtype=t.int32, device="cuda")
        d["starts"] = put(self.starts.astype(np.int32))
        d["slots"] = put(self.slots.astype(np.int32))
        d["mask"] = None if self.mask is None else put(self.mask.view(np.int64))
        d["out"] = self.dev.empty((self.rows, self.q.shape[1]), self.dtype, fill=self.fill)
        d["bytes"] = self.ctx.tree_attn_workspace(rows=self.rows, n_q_heads=self.hq, n_kv_heads=self.hkv, head_dim=self.hd)
        d["work"] = t.full((d["bytes"] + 64,), 255, dtype=t.uint8, device="cuda")  # NaN everywhere: nothing of it is read unwritten
        d["pool"] = L.KvPool(self.ctx, page_rows=self.page, n_pages=self.n_pages, n_slots=self.n_slots, max_pages=self.max_pages, table=d["table"],
                             lens=d["lens"], refs=d["refs"], stores=[d["k"], d["v"]], row_bytes=self.width * d["k"].element_size())
        self.d = d
        return d

    def call(self, stream=None, **over):
        d = self.d
        kw = dict(k_store=0, v_store=1, slots=d["slots"], q_start=d["starts"], n_seqs=len(self.lens), rows=self.rows, mask=d["mask"],
                  mask_words=self.words if d["mask"] is not None else 0, n_q_heads=self.hq, n_kv_heads=self.hkv, head_dim=self.hd, scale=self.scale,
                  dtype=self.dtype, kv_dtype=self.kv, workspace=d["work"], workspace_bytes=d["bytes"], q_row_stride=self.q.shape[1],
                  out_row_stride=self.q.shape[1], stream=stream)
        self.ctx.tree_attn(d["pool"], d["q"], d["out"], **{**kw, **over})

    def run(self):
        self.upload()
        self.call()
        self.ctx.stream_sync()
        return self.dev.get(self.d["out"])

    def check(self, got, what=""):
        g = self.hq // self.hkv
        rounded = self.dtype == self.kv and self.dtype != F32
        for i in range(len(self.lens)):
            n, length = int(self.drafts[i]), int(self.lens[i])
            if n == 0:
                continue
            r0 = int(self.starts[i])
            see = visible(n, length - n, None if self.mask is None else self.mask[r0:r0 + n])
            at = self.cache_row(i, np.arange(length))
            for h in range(self.hq):
                kc = slice((h // g) * self.hd, (h // g + 1) * self.hd)
                qc = slice(h * self.hd, (h + 1) * self.hd)
                out, size, terms = attention(self.q[r0:r0 + n, qc], self.k[at, kc], self.v[at, kc], see, np.float32(self.scale))
                tol = tolerance(out, size, terms, length, self.hd, self.dtype, rounded)
                err = np.abs(got[r0:r0 + n, qc] - out)
                assert (err <= tol).all(), f"{what}: sequence {i}, head {h}: {err.max():.3e} against {tol.flat[np.argmax(err - tol)]:.3e}"
        # nothing else is written: rows behind the last sequence, columns behind the heads
        assert (got[int(self.starts[-1]):] == self.fill).all() and (got[:, self.hq * self.hd:] == self.fill).all(), what


TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (F16, BF16), (BF16, F32)]
RAGGED = dict(lens=[1, 2, 17, 64, 65, 129, 300, 1000], drafts=[1, 2, 5, 9, 1, 33, 12, 20])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", TYPES)
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 64), (14, 2, 64), (4, 2, 128), (2, 1, 256)])
def test_types_and_heads(ctx, dev, dtype, kv, hq, hkv, hd):
    c = Case(ctx, dev, **RAGGED, hq=hq, hkv=hkv, hd=hd, dtype=dtype, kv=kv, seed=hq + hd)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq,hkv,hd", [(3, 3, 40), (6, 2, 72), (5, 1, 80), (20, 1, 96), (34, 2, 64), (150, 1, 64), (2, 2, 1), (3, 1, 5), (1, 1, 130), (4, 4, 192)])
def test_odd_head_sizes_and_groups(ctx, dev, dtype, hq, hkv, hd):
    c = Case(ctx, dev, lens=[1, 40, 200], drafts=[1, 7, 30], hq=hq, hkv=hkv, hd=hd, dtype=dtype, kv=dtype, seed=hd)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", [(F32, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
def test_pages_that_end_anywhere_in_a_tile(ctx, dev, dtype, kv, page, hd):
    c = Case(ctx, dev, lens=[page - 1, page, page + 1, 127, 128, 129, 255, 257, 640], drafts=[1, 1, 2, 3, 4, 5, 6, 65, 130], hq=4, hkv=2, hd=hd, page=page,
             dtype=dtype, kv=kv, seed=page, slots=[3, 0, 7, 1, 2, 5, 4, 9, 6])
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", [(F32, F32), (F32, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("mask", ["chain", "random", "none"])
@pytest.mark.parametrize("hd", [64, 128])
def test_masks(ctx, dev, dtype, kv, mask, hd):
    # "none": drafted rows that see no drafted row, and nothing at all where nothing is committed (rows of zeros)
    c = Case(ctx, dev, lens=[3, 70, 100, 161, 260, 5], drafts=[3, 70, 63, 64, 97, 1], hq=6, hkv=2, hd=hd, dtype=dtype, kv=kv, mask=mask, seed=5)
    got = c.run()
    c.check(got)
    if mask == "none":
        assert (got[:73, :6 * hd] == 0.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", [(F32, F16), (BF16, BF16)])
def test_a_narrow_mask_hides_the_rows_it_has_no_bits_for(ctx, dev, dtype, kv):
    c = Case(ctx, dev, lens=[200], drafts=[150], hq=2, hkv=1, hd=64, dtype=dtype, kv=kv, mask="random", seed=2)
    c.mask, c.words = np.ascontiguousarray(c.mask[:, :1]), 1
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", TYPES)
def test_strides_and_rows_of_no_sequence(ctx, dev, dtype, kv):
    c = Case(ctx, dev, lens=[50, 9, 300], drafts=[3, 0, 17], hq=4, hkv=2, hd=64, dtype=dtype, kv=kv, pad=24, q_pad=40, extra_rows=5, seed=8)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_and_stores_off_the_16_byte_grid(ctx, dev, dtype):
    # strides that are odd, and a q that starts one element into its buffer
    c = Case(ctx, dev, lens=[33, 200], drafts=[2, 9], hq=2, hkv=1, hd=64, dtype=dtype, kv=dtype, pad=2 if dtype == F32 else 1, q_pad=3, seed=9)
    d = c.upload()
    flat = c.torch.zeros(d["q"].numel() + 1, dtype=d["q"].dtype, device="cuda")
    shifted = flat[1:].view(d["q"].shape)
    shifted.copy_(d["q"])
    d["q"] = shifted
    c.call()
    ctx.stream_sync()
    c.check(dev.get(d["out"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(F32, F16, 64), (BF16, BF16, 64), (BF16, BF16, 128), (F16, F16, 128), (F32, F32, 128)])
def test_what_is_not_seen_does_not_reach_a_row(ctx, dev, dtype, kv, hd):
    """Infinities and NaN in rows behind the last position, in pages nobody holds, and in drafted rows that only some see."""
    c = Case(ctx, dev, lens=[150, 41, 300], drafts=[20, 9, 70], hq=4, hkv=2, hd=hd, dtype=dtype, kv=kv, mask="tree", seed=21)
    clean = c.run()
    c.check(clean)
    used = np.zeros(c.n_pages * c.page, bool)
    for i in range(3):
        used[c.cache_row(i, np.arange(int(c.lens[i])))] = True
    c.k[~used], c.v[~used] = np.nan, np.inf
    again = c.run()
    assert np.array_equal(again, clean), "rows that belong to nobody"
    # a drafted row of sequences 0 and 2 goes bad: the rows that do not see it keep their results
    for i, node, kbad, vbad in [(0, 4, 1.0, np.nan), (0, 7, np.nan, 1.0), (2, 30, np.inf, np.inf), (2, 66, 1.0, -np.inf)]:
        row = c.cache_row(i, np.array([int(c.lens[i] - c.drafts[i]) + node]))[0]
        k0, v0 = c.k[row].copy(), c.v[row].copy()
        if kbad != 1.0:
            c.k[row, 3::hd] = kbad
        if vbad != 1.0:
            c.v[row, 3::hd] = vbad
        got = c.run()
        c.k[row], c.v[row] = k0, v0
        r0, n = int(c.starts[i]), int(c.drafts[i])
        sees = visible(n, 0, c.mask[r0:r0 + n])[:, node]
        rows = np.ones(c.rows, bool)
        rows[r0:r0 + n] = ~sees
        # same arithmetic but for the order in which a row's sums are taken: within the tolerance of either
        good = got.copy()
        good[~rows] = clean[~rows]
        c.check(good, f"bad row {node} of sequence {i}")
        hit = got[~rows].reshape(-1, c.hq, hd)
        if vbad != 1.0:
            assert not np.isfinite(hit[:, :, 3]).any()
        if vbad != 1.0 and kbad == 1.0:  # a score of +inf makes the whole row inf - inf
            keep = np.delete(hit, 3, axis=2)
            assert np.isfinite(keep).all()
            assert np.allclose(keep, np.delete(clean[~rows].reshape(-1, c.hq, hd), 3, axis=2), rtol=0.05, atol=0.05)
        if np.isnan(kbad):
            assert np.isnan(hit).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(F32, F16, 64), (F32, F32, 128), (BF16, BF16, 64), (BF16, BF16, 128), (F16, F16, 64)])
def test_long_contexts_are_split_and_joined(ctx, dev, dtype, kv, hd):
    # few rows over many keys: every block of rows is shared by many CTAs
    c = Case(ctx, dev, lens=[20011, 3], drafts=[9, 1], hq=2, hkv=1, hd=hd, page=64, dtype=dtype, kv=kv, seed=31)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(F32, F16, 64), (BF16, BF16, 128), (F16, F16, 64)])
@pytest.mark.parametrize("k_scale", [8.0, 0.0])
def test_large_and_equal_scores(ctx, dev, dtype, kv, hd, k_scale):
    # scores up to some hundred: the running maximum moves often and far; and all equal: every weight is the same
    c = Case(ctx, dev, lens=[700, 90], drafts=[40, 90], hq=4, hkv=2, hd=hd, dtype=dtype, kv=kv, k_scale=k_scale, scale=0.5, seed=41)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(F32, F16, 64), (BF16, BF16, 128), (F16, F16, 64)])
def test_many_sequences(ctx, dev, dtype, kv, hd):
    rng = np.random.default_rng(3)
    n = 300  # more than one pass of the walk's sum takes
    drafts = rng.integers(1, 4, n)
    c = Case(ctx, dev, lens=drafts + rng.integers(0, 200, n), drafts=drafts, hq=2, hkv=1, hd=hd, dtype=dtype, kv=kv, seed=43)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", [(F32, F16), (BF16, BF16)])
def test_bad_sequences_are_reported_and_left_alone(ctx, dev, dtype, kv):
    c = Case(ctx, dev, lens=[50, 60, 70], drafts=[3, 4, 5], hq=4, hkv=2, hd=64, dtype=dtype, kv=kv, seed=51)
    c.run()
    want = dev.get(c.d["out"])
    for change in ("slot", "length", "rows"):
        d = c.upload()
        if change == "slot":
            d["slots"][1] = 99
        elif change == "length":
            d["lens"][1] = 3  # fewer positions than drafted rows
        else:
            d["starts"][3] = 13  # one row more than the call has
        c.call()
        with pytest.raises(L.LokalCudaError) as e:
            ctx.stream_sync()
        assert e.value.status == capi.ERR_PAGE_RANGE
        got, lost = dev.get(d["out"]), slice(3, 7) if change != "rows" else slice(7, 12)
        assert (got[lost] == c.fill).all()
        keep = np.ones(12, bool)
        keep[lost] = False
        assert np.allclose(got[keep], want[keep], rtol=2e-2, atol=2e-2) and (got[keep] != c.fill).any()
    # a page that is not there: reported, nothing outside the pool is read
    d = c.upload()
    d["table"][1, 1] = -1
    d["table"][2, 0] = 1 << 30
    c.call()
    with pytest.raises(L.LokalCudaError) as e:
        ctx.stream_sync()
    assert e.value.status == capi.ERR_PAGE_RANGE
    assert np.allclose(dev.get(d["out"])[:3], want[:3], rtol=2e-2, atol=2e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", [(F32, F16), (BF16, BF16)])
def test_captured_and_on_two_streams(ctx, dev, dtype, kv):
    a = Case(ctx, dev, lens=[500, 1200], drafts=[8, 30], hq=4, hkv=2, hd=64, dtype=dtype, kv=kv, seed=61)
    b = Case(ctx, dev, lens=[90], drafts=[3], hq=4, hkv=2, hd=64, dtype=dtype, kv=kv, seed=62)
    first, second = a.run(), b.run()
    s, t = ctx.stream_create(), ctx.stream_create()
    a.torch.cuda.synchronize()
    ctx.graph_begin(s)
    a.call(stream=s)
    graph = ctx.graph_end(s)
    for _ in range(5):
        a.d["out"].fill_(0.0)
        b.d["out"].fill_(0.0)
        a.torch.cuda.synchronize()
        ctx.graph_launch(graph, s)
        b.call(stream=t)
        ctx.stream_sync(s)
        ctx.stream_sync(t)
        assert np.array_equal(dev.get(a.d["out"])[:, :256], first[:, :256]) and np.array_equal(dev.get(b.d["out"])[:, :256], second[:, :256])
    # the lengths are read when the graph runs: a shorter sequence, same graph
    a.lens[1] = 700
    a.d["lens"].copy_(dev.put(np.array([500, 700, 0], np.int32)))
    a.torch.cuda.synchronize()
    ctx.graph_launch(graph, s)
    ctx.stream_sync(s)
    a.fill = 0.0
    a.check(dev.get(a.d["out"]))
    ctx.graph_destroy(graph)
    ctx.stream_destroy(s)
    ctx.stream_destroy(t)


@pytest.mark.gpu
def test_refusals(ctx, dev):
    c = Case(ctx, dev, lens=[50], drafts=[3], hq=4, hkv=2, hd=64, dtype=BF16, kv=BF16, seed=71)
    d = c.upload()
    for over, status in [(dict(k_store=2), capi.ERR_BAD_ARG), (dict(dtype=L.Q8_0), capi.ERR_UNSUPPORTED), (dict(kv_dtype=L.Q8_0), capi.ERR_UNSUPPORTED),
                         (dict(n_q_heads=5), capi.ERR_BAD_ARG), (dict(n_kv_heads=0), capi.ERR_BAD_ARG), (dict(head_dim=0), capi.ERR_BAD_ARG),
                         (dict(head_dim=257, n_kv_heads=1, n_q_heads=1), capi.ERR_UNSUPPORTED), (dict(n_kv_heads=4), capi.ERR_BAD_ARG),
                         (dict(kv_dtype=F32), capi.ERR_BAD_ARG), (dict(mask_words=0), capi.ERR_BAD_ARG), (dict(q_row_stride=255), capi.ERR_BAD_ARG),
                         (dict(out_row_stride=1), capi.ERR_BAD_ARG), (dict(workspace=None), capi.ERR_BAD_ARG),
                         (dict(workspace_bytes=d["bytes"] - 1), capi.ERR_BAD_ARG), (dict(workspace=d["work"].data_ptr() + 8), capi.ERR_MISALIGNED),
                         (dict(q_start=None), capi.ERR_BAD_ARG), (dict(mask=d["mask"].data_ptr() + 4), capi.ERR_MISALIGNED)]:
        with pytest.raises(L.LokalCudaError) as e:
            c.call(**over)
        assert e.value.status == status, over
    for x in ("q", "out"):
        with pytest.raises(L.LokalCudaError) as e:
            ctx.tree_attn(d["pool"], d["q"].data_ptr() + (x == "q"), d["out"].data_ptr() + (x == "out"), k_store=0, v_store=1, q_start=d["starts"], n_seqs=1,
                          rows=3, n_q_heads=4, n_kv_heads=2, head_dim=64, scale=1.0, dtype=BF16, kv_dtype=BF16, workspace=d["work"], workspace_bytes=d["bytes"])
        assert e.value.status == capi.ERR_MISALIGNED
    c.call(n_seqs=0)
    c.call(rows=0)
    ctx.stream_sync()
    assert (dev.get(d["out"]) == c.fill).all(), "a refused or empty call writes nothing"
    assert ctx.tree_attn_workspace(rows=3, n_q_heads=4, n_kv_heads=2, head_dim=300) == 0


# ---- the plan ----

@pytest.mark.gpu
@pytest.mark.parametrize("chain", [False, True])
def test_plan_follows_the_parents(ctx, dev, chain):
    import torch
    c = Case(ctx, dev, lens=[9, 300, 131, 70], drafts=[9, 200, 0, 65], hq=1, hkv=1, hd=8, seed=81, extra_rows=3)
    rng = np.random.default_rng(1)
    parents = [np.arange(n) - 1 if chain else random_parents(rng, int(n)) for n in c.drafts]
    d = c.upload()
    words = 4
    mask = torch.full((c.rows, words), -1, dtype=torch.int64, device="cuda")
    pos = torch.full((c.rows,), -9, dtype=torch.int32, device="cuda")
    rows = torch.full((c.rows,), -9, dtype=torch.int32, device="cuda")
    up = None if chain else dev.put(np.concatenate([*parents, np.zeros(3)]).astype(np.int32))
    ctx.tree_plan(d["pool"], q_start=d["starts"], slots=d["slots"], n_seqs=4, rows=c.rows, parents=up, mask=mask, mask_words=words, positions=pos,
                  cache_rows=rows)
    ctx.stream_sync()
    mask, pos, rows = mask.cpu().numpy().view(np.uint64), pos.cpu().numpy(), rows.cpu().numpy()
    for i, p in enumerate(parents):
        r0, n, base = int(c.starts[i]), len(p), int(c.lens[i] - c.drafts[i])
        depth = np.zeros(n, int)
        for j, a in enumerate(p):
            depth[j] = depth[a] + 1 if a >= 0 else 0
        assert np.array_equal(mask[r0:r0 + n], mask_of(p, words))
        assert np.array_equal(pos[r0:r0 + n], base + depth)
        assert np.array_equal(rows[r0:r0 + n], c.cache_row(i, base + np.arange(n)))
    assert (mask[-3:] == np.uint64(2 ** 64 - 1)).all() and (pos[-3:] == -9).all() and (rows[-3:] == -9).all()


@pytest.mark.gpu
def test_plan_reports_bad_parents_and_narrow_masks(ctx, dev):
    import torch
    c = Case(ctx, dev, lens=[80], drafts=[70], hq=1, hkv=1, hd=8, seed=82)
    d = c.upload()
    mask = torch.zeros((70, 2), dtype=torch.int64, device="cuda")
    parents = random_parents(np.random.default_rng(2), 70)
    for j, bad in ((5, 5), (6, 40), (7, -2), (0, 3)):
        p = parents.copy()
        p[j] = bad
        ctx.tree_plan(d["pool"], q_start=d["starts"], n_seqs=1, rows=70, parents=dev.put(p), mask=mask, mask_words=2)
        with pytest.raises(L.LokalCudaError) as e:
            ctx.stream_sync()
        assert e.value.status == capi.ERR_PAGE_RANGE
        p[j] = -1
        assert np.array_equal(mask.cpu().numpy().view(np.uint64), mask_of(p, 2))
    ctx.tree_plan(d["pool"], q_start=d["starts"], n_seqs=1, rows=70, parents=dev.put(parents), mask=mask, mask_words=1)
    with pytest.raises(L.LokalCudaError) as e:
        ctx.stream_sync()
    assert e.value.status == capi.ERR_PAGE_RANGE
    for kw in (dict(mask_words=0), dict(q_start=None)):
        with pytest.raises(L.LokalCudaError) as e:
            ctx.tree_plan(d["pool"], **{**dict(q_start=d["starts"], n_seqs=1, rows=70, mask=mask, mask_words=1), **kw})
        assert e.value.status == capi.ERR_BAD_ARG


# ---- all of it together ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", [(BF16, BF16), (F32, F16)])
def test_draft_verify_accept_steps(ctx, dev, dtype, kv):
    """Two prompts, one forked, then steps of: grow, plan, rotate K into the cache, stage V, attend, accept a path, compact. The
    attention of every step agrees with a plain one over the rows that each sequence should hold by then."""
    import torch
    cfg = synth.LayerConfig("steps", dtype, 64, 64, 64, 4, 2, 64, 100, 1e4, 1e-6, 1, seed=90)
    hq, hkv, hd, page, n_pages, n_slots = 4, 2, 64, 16, 60, 4
    width = hkv * hd
    rng = np.random.default_rng(17)
    put = dev.put
    ints = lambda a: put(np.asarray(a, np.int32))
    kstore, vstore = dev.empty((n_pages * page, width), kv, fill=3.0), dev.empty((n_pages * page, width), kv, fill=3.0)
    table, lens, refs = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((n_slots, 20), (n_slots,), (n_pages,)))
    pool = L.KvPool(ctx, page_rows=page, n_pages=n_pages, n_slots=n_slots, max_pages=20, table=table, lens=lens, refs=refs, stores=[kstore, vstore],
                    row_bytes=width * kstore.element_size())
    pool.reset()
    held = {}  # slot -> list of (k row, v row) as the cache should hold them

    def stage(slots, n_rows, parents):
        """Grows, plans and stages; returns what the attention call needs."""
        starts = np.concatenate([[0], np.cumsum(n_rows)])
        rows, words = int(starts[-1]), -(-max(n_rows) // 64)
        dslots, dstarts = ints(slots), ints(starts)
        pool.reserve(dslots, ints([len(held[s]) + n for s, n in zip(slots, n_rows)]), n=len(slots))
        mask = torch.zeros((rows, words), dtype=torch.int64, device="cuda") if parents is not None else None
        pos, crow = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
        up = None if parents is None else ints(np.concatenate(parents))
        ctx.tree_plan(pool, slots=dslots, q_start=dstarts, n_seqs=len(slots), rows=rows, parents=up, mask=mask, mask_words=words if mask is not None else 0,
                      positions=pos, cache_rows=crow)
        q, k, v = (synth.round_to(rng.standard_normal((rows, w), dtype=np.float32), dtype) for w in (hq * hd, width, width))
        dq, dk, dv = put(q, dtype), put(k, dtype), put(v, dtype)
        rope = torch.zeros((rows, hd), dtype=torch.float32, device="cuda")
        ctx.rope_table(rope, theta=cfg.theta, rot_dim=hd, rows=rows, positions=pos)
        p = ctx.qk_rope_params(q=dq, k=dk, k_out=dk, cos_sin=rope, rows=rows, n_q_heads=hq, n_kv_heads=hkv, head_dim=hd, q_dtype=dtype, k_dtype=dtype, w_dtype=F32)
        ctx.qk_rope(p)
        for src, dst in ((dk, kstore), (dv, vstore)):
            ctx.kv_stage(src, dst, src_dtype=dtype, dst_dtype=kv, rows=rows, width=width, dst_rows=crow)
        ctx.stream_sync()
        kk, vv = synth.round_to(dev.get(dk), kv), synth.round_to(v, kv)
        return starts, mask, dq, kk, vv, dslots, dstarts, rows, words

    def attend_and_check(slots, n_rows, made):
        starts, mask, dq, kk, vv, dslots, dstarts, rows, words = made
        out = dev.empty((rows, hq * hd), dtype, fill=0.0)
        nbytes = ctx.tree_attn_workspace(rows=rows, n_q_heads=hq, n_kv_heads=hkv, head_dim=hd)
        work = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        ctx.tree_attn(pool, dq, out, k_store=0, v_store=1, slots=dslots, q_start=dstarts, n_seqs=len(slots), rows=rows, mask=mask,
                      mask_words=words if mask is not None else 0, n_q_heads=hq, n_kv_heads=hkv, head_dim=hd, scale=hd ** -0.5, dtype=dtype, kv_dtype=kv,
                      workspace=work, workspace_bytes=nbytes)
        ctx.stream_sync()
        got, q = dev.get(out), dev.get(dq)
        bits_ = None if mask is None else mask.cpu().numpy().view(np.uint64)
        for i, s in enumerate(slots):
            r0, n = int(starts[i]), n_rows[i]
            ks = np.concatenate([np.array([a for a, _ in held[s]], np.float32).reshape(-1, width), kk[r0:r0 + n]])
            vs = np.concatenate([np.array([b for _, b in held[s]], np.float32).reshape(-1, width), vv[r0:r0 + n]])
            see = visible(n, len(held[s]), None if bits_ is None else bits_[r0:r0 + n])
            for h in range(hq):
                kc, qc = slice(h // 2 * hd, (h // 2 + 1) * hd), slice(h * hd, (h + 1) * hd)
                o, size, terms = attention(q[r0:r0 + n, qc], ks[:, kc], vs[:, kc], see, np.float32(hd ** -0.5))
                assert (np.abs(got[r0:r0 + n, qc] - o) <= tolerance(o, size, terms, len(ks), hd, dtype, dtype == kv)).all()

    # prompts, as chains
    held[0], held[1] = [], []
    made = stage([0, 1], [37, 90], None)
    attend_and_check([0, 1], [37, 90], made)
    for s, r0, n in ((0, 0, 37), (1, 37, 90)):
        held[s] = [(made[3][r0 + j], made[4][r0 + j]) for j in range(n)]
    pool.fork(ints([1]), ints([2]), n=1)
    held[2] = list(held[1])
    for step in range(4):
        slots = [0, 1, 2]
        n_rows = [int(x) for x in rng.integers(1, 40, 3)]
        parents = [random_parents(rng, n) for n in n_rows]
        made = stage(slots, n_rows, parents)
        attend_and_check(slots, n_rows, made)
        # one path from a child of the last committed row down
        acc, counts = np.zeros((3, 8), np.int32), []
        for i in range(3):
            path, at = [], -1
            while len(path) < 8:
                children = [j for j in range(n_rows[i]) if parents[i][j] == at]
                if not children:
                    break
                at = int(rng.choice(children))
                path.append(at)
            acc[i, :len(path)] = path
            counts.append(len(path))
            held[slots[i]] += [(made[3][made[0][i] + j], made[4][made[0][i] + j]) for j in path]
        pool.accept(made[5], made[6], ints(acc.reshape(-1)), ints(counts), n_seqs=3, max_accept=8)
        if step == 1:
            pool.truncate(ints([0]), n=1)
            held[0] = []
        if step % 2:
            pool.compact()
        ctx.stream_sync()
        assert list(lens.cpu().numpy()[:3]) == [len(held[s]) for s in slots]
    pool.close()


# ---- what only large or unusual calls reach ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F16, 64), (F32, 128)])
def test_rows_past_four_gigabytes(ctx, dev, dtype, hd):
    """Pages at the far end of a store of 5 GB (one store is K and V at once): byte offsets need more than 32 bits."""
    import torch
    hkv, page = 8, 64
    c = Case(ctx, dev, lens=[300, 70], drafts=[9, 70], hq=8, hkv=hkv, hd=hd, page=page, dtype=dtype, kv=dtype, seed=101)
    row_bytes = hkv * hd * (4 if dtype == F32 else 2)
    far = 5 * 2 ** 30 // (page * row_bytes)
    d = c.upload()
    big = torch.empty(((far + c.n_pages) * page, hkv * hd), dtype=d["k"].dtype, device="cuda")
    big[far * page:] = d["k"]
    c.v = c.k
    pool = L.KvPool(ctx, page_rows=page, n_pages=far + c.n_pages, n_slots=c.n_slots, max_pages=c.max_pages, table=d["table"] + far * (d["table"] >= 0).int(),
                    lens=d["lens"], refs=torch.zeros(far + c.n_pages, dtype=torch.int32, device="cuda"), stores=[big], row_bytes=row_bytes)
    ctx.tree_attn(pool, d["q"], d["out"], k_store=0, v_store=0, slots=d["slots"], q_start=d["starts"], n_seqs=2, rows=c.rows, mask=d["mask"],
                  mask_words=c.words, n_q_heads=8, n_kv_heads=hkv, head_dim=hd, scale=c.scale, dtype=dtype, kv_dtype=dtype, workspace=d["work"],
                  workspace_bytes=d["bytes"])
    ctx.stream_sync()
    c.check(dev.get(d["out"]))
    # and pages are copied there and back
    pair = lambda *x: dev.put(np.array(x, np.int32))
    pool.copy_pages(pair(far, far + 1), pair(0, far + c.n_pages - 1), n=2)
    ctx.stream_sync()
    assert torch.equal(big[:page], big[far * page:(far + 1) * page])
    assert torch.equal(big[-page:], big[(far + 1) * page:(far + 2) * page])
    pool.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(BF16, BF16, 64), (F16, F16, 128), (F32, F16, 128), (F32, F32, 64)])
def test_more_sequences_than_a_walk_remembers(ctx, dev, dtype, kv, hd):
    # thousands of short sequences: each CTA steps through more of them than fit its shared memory, and a block is one tile
    rng = np.random.default_rng(7)
    n = 6000
    drafts = rng.integers(0, 3, n)
    drafts[0] = 2
    c = Case(ctx, dev, lens=drafts + rng.integers(1, 20, n), drafts=drafts, hq=2, hkv=1, hd=hd, page=8, dtype=dtype, kv=kv, seed=103)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(BF16, BF16, 64), (BF16, BF16, 128), (F32, F16, 64)])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales_that_are_negative_or_zero(ctx, dev, dtype, kv, hd, scale):
    c = Case(ctx, dev, lens=[200, 33], drafts=[7, 33], hq=4, hkv=2, hd=hd, dtype=dtype, kv=kv, scale=scale, seed=105)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [120, 128, 129, 300])
def test_sequences_with_more_drafted_rows_than_a_tile(ctx, dev, drafts):
    # masks of two words and of more, trees that reach over several key tiles and blocks of rows
    for dtype in (BF16, F32):
        c = Case(ctx, dev, lens=[drafts + 61, drafts], drafts=[drafts, drafts], hq=6, hkv=2, hd=64, dtype=dtype, kv=dtype, mask="tree", seed=drafts)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_a_wait_that_runs_out_is_an_error_and_the_next_call_is_right(ctx, dev, monkeypatch, hd):
    # the copies announce 16 bytes more than they bring (as in tests/test_gpu_timeout.py): every wait for one gives up
    c = Case(ctx, dev, lens=[3000, 500], drafts=[9, 5], hq=4, hkv=2, hd=hd, dtype=BF16, kv=BF16, seed=107)
    c.upload()
    monkeypatch.setenv("LOKAL_CUDA_TEST_EXTRA_TX", "16")
    monkeypatch.setenv("LOKAL_CUDA_WAIT_LIMIT", "200")
    c.call()
    with pytest.raises(L.LokalCudaError) as e:
        ctx.stream_sync()
    assert e.value.status == capi.ERR_TIMEOUT
    monkeypatch.delenv("LOKAL_CUDA_WAIT_LIMIT")
    monkeypatch.delenv("LOKAL_CUDA_TEST_EXTRA_TX")
    c.d["out"].fill_(c.fill)
    c.call()
    ctx.stream_sync()
    c.check(dev.get(c.d["out"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(BF16, BF16, 128), (F16, F16, 64), (F32, F16, 64), (F32, F32, 40)])
def test_the_same_bits_every_time(ctx, dev, dtype, kv, hd):
    c = Case(ctx, dev, lens=[5000, 900, 77], drafts=[20, 3, 40], hq=4, hkv=2, hd=hd, dtype=dtype, kv=kv, seed=109)
    first = c.run()
    for _ in range(5):
        c.call()
        ctx.stream_sync()
        assert np.array_equal(dev.get(c.d["out"]), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("mask", ["tree", "random", None])
def test_sequences_of_few_rows_beside_some_of_many(ctx, dev, dtype, mask):
    """Head size 64 with few rows to a sequence on average: blocks of up to 16 rows and larger ones (and the short last block of a
    long sequence), in any order, of one key tile and of many."""
    rng = np.random.default_rng(113)
    drafts = rng.integers(0, 8, 40)
    drafts[[3, 4, 17, 30]] = [65, 40, 70, 9]
    lens = drafts + rng.choice([0, 1, 90, 128, 700, 2500], 40)
    lens[drafts == 0] += 1
    assert drafts.sum() * 2 <= 16 * 40
    c = Case(ctx, dev, lens=lens, drafts=drafts, hq=6, hkv=3, hd=64, dtype=dtype, kv=dtype, mask=mask, seed=114)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd", [(8, 4, 64), (32, 2, 64), (2, 2, 64), (8, 4, 128)])
def test_single_tokens_of_many_long_sequences(ctx, dev, hq, hkv, hd):
    rng = np.random.default_rng(115)
    n = 96
    c = Case(ctx, dev, lens=rng.integers(1, 4000, n), drafts=np.ones(n, np.int64), hq=hq, hkv=hkv, hd=hd, dtype=BF16, kv=BF16, mask=None, seed=116)
    first = c.run()
    c.check(first)
    for _ in range(5):
        assert np.array_equal(c.run(), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(F16, F16, 64), (BF16, BF16, 64), (F16, F16, 128), (F32, F16, 64)])
def test_what_few_rows_do_not_see_does_not_reach_them(ctx, dev, dtype, kv, hd):
    """As above with short sequences, where the rows that see a bad value would show the loss of the key's other columns."""
    c = Case(ctx, dev, lens=[150, 8, 131], drafts=[6, 8, 5], hq=4, hkv=2, hd=hd, dtype=dtype, kv=kv, mask="tree", seed=117)
    clean = c.run()
    c.check(clean)
    used = np.zeros(c.n_pages * c.page, bool)
    for i in range(3):
        used[c.cache_row(i, np.arange(int(c.lens[i])))] = True
    c.k[~used], c.v[~used] = np.nan, np.inf
    assert np.array_equal(c.run(), clean), "rows that belong to nobody"
    for i, node, bad in [(0, 2, np.nan), (1, 3, np.inf), (2, 3, -np.inf)]:
        row = c.cache_row(i, np.array([int(c.lens[i] - c.drafts[i]) + node]))[0]
        before = c.v[row].copy()
        c.v[row, 3::hd] = bad
        got = c.run()
        c.v[row] = before
        r0, n = int(c.starts[i]), int(c.drafts[i])
        rows = np.zeros(c.rows, bool)
        rows[r0:r0 + n] = visible(n, 0, c.mask[r0:r0 + n])[:, node]
        good = got.copy()
        good[rows] = clean[rows]
        c.check(good, f"bad row {node} of sequence {i}")
        hit, was = got[rows].reshape(-1, c.hq, hd), clean[rows].reshape(-1, c.hq, hd)
        assert rows.any() and not np.isfinite(hit[:, :, 3]).any()
        # two results of the same formula, each within its tolerance (values of order 1): 2 * 2^-8 of the largest, and to spare
        assert np.allclose(np.delete(hit, 3, axis=2), np.delete(was, 3, axis=2), rtol=0.05, atol=0.05)


@pytest.mark.gpu
def test_out_is_not_q(ctx, dev):
    c = Case(ctx, dev, lens=[50], drafts=[3], hq=4, hkv=2, hd=64, dtype=BF16, kv=BF16, seed=119)
    d = c.upload()
    d["out"] = d["q"]
    with pytest.raises(L.LokalCudaError) as e:
        c.call()
    assert e.value.status == capi.ERR_BAD_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,drafts,hd", [(BF16, 1, 64), (F16, 40, 64), (BF16, 1, 128)])
def test_the_first_query_rows_of_a_cta_come_through_whole(ctx, dev, dtype, drafts, hd):
    """The tile they are copied into is where the walk to a CTA's share keeps its sums before: two calls in turn, many times, with
    other query rows and so another walk's sums under them."""
    n = 300
    cases = [Case(ctx, dev, lens=np.full(n, 150 + 60 * i), drafts=np.full(n, drafts), hq=4, hkv=2, hd=hd, dtype=dtype, kv=dtype, mask=None, seed=121 + i) for i in range(2)]
    first = [c.run() for c in cases]
    for c, got in zip(cases, first):
        c.check(got)
    for _ in range(100):
        for c in cases:
            c.call()
    ctx.stream_sync()
    for c, got in zip(cases, first):
        assert np.array_equal(dev.get(c.d["out"]), got)


# ---- infinities and the largest numbers in what is seen ----

def seen_by(c, i):
    n, length = int(c.drafts[i]), int(c.lens[i])
    r0 = int(c.starts[i])
    return visible(n, length - n, None if c.mask is None else c.mask[r0:r0 + n])


def check_columns(c, got, columns, see, k=None, v=None):
    """The given columns of every head against the f64 form, with `see[i]` for what the rows of sequence i see and, where given,
    other K and V than the cache's."""
    g, rounded = c.hq // c.hkv, c.dtype == c.kv and c.dtype != F32
    k, v = c.k if k is None else k, c.v if v is None else v
    for i in range(len(c.lens)):
        n, length, r0 = int(c.drafts[i]), int(c.lens[i]), int(c.starts[i])
        at = c.cache_row(i, np.arange(length))
        for h in range(c.hq):
            kc, qc = slice(h // g * c.hd, (h // g + 1) * c.hd), slice(h * c.hd, (h + 1) * c.hd)
            out, size, terms = attention(c.q[r0:r0 + n, qc], k[at, kc], v[at, kc], see[i], np.float32(c.scale))
            tol = tolerance(out, size, terms, length, c.hd, c.dtype, rounded)
            bad = ~(np.abs(got[r0:r0 + n, qc] - out) <= tol)[:, columns]
            assert not bad.any(), f"sequence {i}, head {h}: {bad.sum()} of {bad.size}"


EVERY_PAIR = [(F32, F32, 64), (F32, F16, 64), (F32, BF16, 64), (F16, F32, 64), (F16, BF16, 64), (BF16, F16, 64), (F16, F16, 64), (BF16, BF16, 64),
              (F32, F32, 128), (F32, F16, 128), (BF16, F32, 128), (F16, F16, 128), (BF16, BF16, 128), (F32, F16, 40), (F16, F16, 40)]


def three_sequences(ctx, dev, dtype, kv, hd, seed):
    return Case(ctx, dev, lens=[150, 41, 2500], drafts=[6, 9, 3], hq=4, hkv=2, hd=hd, dtype=dtype, kv=kv, seed=seed)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", EVERY_PAIR)
def test_a_key_with_a_score_of_minus_infinity_weighs_nothing(ctx, dev, dtype, kv, hd):
    """Committed and drafted keys with one element of -inf that all query rows meet with a positive number: exactly the result
    without these keys."""
    c = three_sequences(ctx, dev, dtype, kv, hd, 131)
    column = np.abs(c.q[:, 5::hd]) + np.float32(0.25)
    column[::2] = 1.0  # and one that any shorter type holds exactly
    c.q[:, 5::hd] = synth.round_to(column, dtype)
    see = [seen_by(c, i) for i in range(3)]
    for i, pos in [(0, 3), (0, 70), (0, 146), (1, 0), (1, 33), (2, 127), (2, 128), (2, 1900), (2, 2497)]:
        c.k[c.cache_row(i, np.array([pos]))[0], 5::hd] = -np.inf
        see[i][:, pos] = False
    got = c.run()
    check_columns(c, got, np.ones(hd, bool), see, k=np.where(np.isfinite(c.k), c.k, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", EVERY_PAIR)
def test_an_infinite_value_in_a_committed_row_is_the_result_of_its_column(ctx, dev, dtype, kv, hd):
    c = three_sequences(ctx, dev, dtype, kv, hd, 133)
    for i, pos, column, value in [(0, 20, 3, np.inf), (0, 21, 9, -np.inf), (1, 31, 3, -np.inf), (2, 5, 9, np.inf), (2, 2300, 3, np.inf),
                                  (2, 700, 20, np.inf), (2, 1500, 20, -np.inf)]:
        c.v[c.cache_row(i, np.array([pos]))[0], column::hd] = value
    got = c.run()
    by_head = got[:, :c.hq * hd].reshape(-1, c.hq, hd)
    s = [slice(int(c.starts[i]), int(c.starts[i + 1])) for i in range(3)]
    assert (by_head[s[0], :, 3] == np.inf).all() and (by_head[s[0], :, 9] == -np.inf).all()
    assert (by_head[s[1], :, 3] == -np.inf).all()
    assert (by_head[s[2], :, 9] == np.inf).all() and (by_head[s[2], :, 3] == np.inf).all()
    assert np.isnan(by_head[s[2], :, 20]).all()  # one of either sign
    columns = np.ones(hd, bool)
    columns[[3, 9, 20]] = False
    see = [seen_by(c, i) for i in range(3)]
    check_columns(c, got, columns, see, v=np.where(np.isfinite(c.v), c.v, 0))
    for i in (0, 1):  # their other columns are as good as ever
        assert np.isfinite(by_head[s[i]][:, :, [20] + ([9] if i else [])]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv,hd", [(F32, F32, 64), (F32, F32, 128), (F32, F16, 64), (F32, BF16, 128), (F16, F32, 64), (BF16, F32, 128), (F32, F32, 40)])
def test_the_largest_numbers_of_32_bits(ctx, dev, dtype, kv, hd):
    """They round up to an infinity in shorter types. A key's meets query elements of 2e-38 (a score of some units), a query's keys of
    0, a value's is weighed down to a finite result."""
    most = np.finfo(np.float32).max
    c = three_sequences(ctx, dev, dtype, kv, hd, 135)
    if kv == F32:
        c.q[:, 5::hd] = synth.round_to(np.full_like(c.q[:, 5::hd], 2e-38), dtype)  # 0 in f16
        for i, pos in [(0, 10), (1, 38), (2, 2000)]:
            c.k[c.cache_row(i, np.array([pos]))[0], 5::hd] = -most
            c.v[c.cache_row(i, np.array([pos + 1]))[0], 7::hd] = most
    if dtype == F32:
        c.q[:, 11::hd] = most
        c.k[:, 11::hd] = 0.0
    got = c.run()
    # a result above the largest number of a 16-bit row type is an infinity there: the column is looked at only in f32 and bf16
    columns = np.ones(hd, bool)
    columns[7] = dtype != F16
    check_columns(c, got, columns, [seen_by(c, i) for i in range(3)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("drafts,hd", [(1, 64), (40, 64), (40, 128)])
@pytest.mark.parametrize("nats", [9.0, 17.0, 20.0])
def test_many_small_weights_beside_large_ones(ctx, dev, dtype, drafts, hd, nats):
    """Eight keys, one in every 32 of the first two tiles, that weigh exp(nats) times as much as each of 100,000 others, and whose
    values are 0: the result is what the others' weights add up to, 60 % to 0.003 % of all. As many sequences as the GPU has SMs hold
    the same pages, so that a CTA has all keys of one and meets the large weights first.

    A weight of f16 loses bits below 2^-14 of what it is rounded at. The kernel takes weights times 2^11 and the largest as 1 or
    more, so what is lost is half a step of 2^-24, 2^-36 of the largest weight; against a sum of at least that weight it is
    keys * 2^-36 of the largest value."""
    import torch
    n, sms = 100000, torch.cuda.get_device_properties(0).multi_processor_count
    c = Case(ctx, dev, lens=[n + drafts], drafts=[drafts], hq=2, hkv=1, hd=hd, page=64, dtype=dtype, kv=dtype, mask="none", seed=141, scale=0.125)
    c.q[:] = 8.0
    c.k[:] = 0.0
    c.v[:] = synth.round_to(1.0 + 0.25 * c.v, dtype)
    large = c.cache_row(0, np.arange(8) * 32 + 5)
    c.k[large, 0], c.v[large] = nats, 0.0
    d = c.upload()
    table = d["table"][:1].repeat(sms, 1).contiguous()
    lens = torch.full((sms,), n + drafts, dtype=torch.int32, device="cuda")
    starts = torch.arange(sms + 1, dtype=torch.int32, device="cuda") * drafts
    q, mask, out = d["q"].repeat(sms, 1), d["mask"].repeat(sms, 1), d["out"].repeat(sms, 1)
    pool = L.KvPool(ctx, page_rows=64, n_pages=c.n_pages, n_slots=sms, max_pages=c.max_pages, table=table, lens=lens, refs=d["refs"], stores=[d["k"], d["v"]],
                    row_bytes=2 * hd)
    ctx.tree_attn(pool, q, out, k_store=0, v_store=1, q_start=starts, n_seqs=sms, rows=sms * drafts, mask=mask, mask_words=c.words, n_q_heads=2, n_kv_heads=1,
                  head_dim=hd, scale=c.scale, dtype=dtype, kv_dtype=dtype, workspace=d["work"], workspace_bytes=d["bytes"])
    ctx.stream_sync()
    pool.close()
    rows = c.cache_row(0, np.arange(n))
    want, size, terms = attention(c.q[:1, :hd], c.k[rows], c.v[rows], np.ones((1, n), bool), np.float32(c.scale))
    tol = tolerance(want, size, terms, n, hd, dtype, True) + n * 2.0 ** -36 * np.abs(c.v).max()
    err = np.abs(dev.get(out).reshape(-1, hd) - want)
    assert (err <= tol).all(), f"{err.max():.3e} of {np.abs(want).max():.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [8, 30])
def test_slots_past_two_to_the_thirty(ctx, dev, drafts):
    """Infinities in a drafted V row are added by way of the page table: its row is that of the slot, not of another one that has the
    same low bits."""
    import torch
    c = Case(ctx, dev, lens=[40, 40], drafts=[drafts, drafts], hq=2, hkv=1, hd=64, page=64, dtype=BF16, kv=BF16, mask=None, seed=151)
    c.v[c.cache_row(0, np.array([40 - drafts]))[0], 5] = np.inf  # the first drafted row, which all see
    want = c.run()
    slots = 2 ** 30 + 4
    table = torch.empty((slots, 1), dtype=torch.int32, device="cuda")
    lens = torch.empty(slots, dtype=torch.int32, device="cuda")
    for at, i in ((slots - 2, 0), (2, 1)):  # 2^30 + 2 and 2
        table[at, 0], lens[at] = int(c.table[i, 0]), 40
    d = c.d
    pool = L.KvPool(ctx, page_rows=64, n_pages=c.n_pages, n_slots=slots, max_pages=1, table=table, lens=lens, refs=d["refs"], stores=[d["k"], d["v"]],
                    row_bytes=128)
    d["out"].fill_(c.fill)
    ctx.tree_attn(pool, d["q"], d["out"], k_store=0, v_store=1, slots=dev.put(np.array([slots - 2, 2], np.int32)), q_start=d["starts"], n_seqs=2, rows=c.rows,
                  n_q_heads=2, n_kv_heads=1, head_dim=64, scale=c.scale, dtype=BF16, kv_dtype=BF16, workspace=d["work"], workspace_bytes=d["bytes"])
    ctx.stream_sync()
    pool.close()
    got = dev.get(d["out"])
    assert (want[:drafts, 5::64] == np.inf).all() and np.isfinite(want[drafts:]).all()
    assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,hd,drafts", [(14, 2, 128, 40), (14, 2, 64, 40), (100, 1, 128, 3), (100, 1, 64, 3), (2, 1, 64, 2)])
def test_rows_of_a_tile_that_are_nobodys_change_no_bit(ctx, dev, dtype, hq, hkv, hd, drafts):
    """A tile of 128 query rows holds as many as divide by the query heads to a key head. What lies in the rest is what an earlier
    call left there, here one with large scores. Nor do the rows of other sequences that share a tile matter."""
    n = 160
    c = Case(ctx, dev, lens=np.full(n, 700), drafts=np.full(n, drafts), hq=hq, hkv=hkv, hd=hd, dtype=dtype, kv=dtype, mask=None, seed=161)
    other = Case(ctx, dev, lens=np.full(n, 300), drafts=np.full(n, drafts), hq=hq // hkv, hkv=1, hd=hd, dtype=dtype, kv=dtype, mask=None, seed=162)
    other.q *= 64.0
    big = Case(ctx, dev, lens=np.full(n, 300), drafts=np.full(n, 128), hq=1, hkv=1, hd=hd, dtype=dtype, kv=dtype, mask=None, seed=163)
    big.q *= 64.0
    first = c.run()
    other.upload()
    big.upload()
    for _ in range(5):
        other.call()
        big.call()
        c.call()
        ctx.stream_sync()
        assert np.array_equal(dev.get(c.d["out"]), first)
    # every second sequence's rows with scores 64 times as large: the others' results stay
    c.d["q"].view(n, drafts, -1)[::2] *= 64.0
    c.call()
    ctx.stream_sync()
    again = dev.get(c.d["out"]).reshape(n, -1)
    assert np.array_equal(again[1::2], first.reshape(n, -1)[1::2])
