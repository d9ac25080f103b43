"""Eviction by accumulated attention weight, through the C ABI: lists, counts, scores and every byte of the cache are
compared for equality with a plain form in numpy; nothing here has a tolerance."""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R

pytestmark = pytest.mark.gpu


def _scores(kind, rng, shape):
    x = rng.random(shape)
    if kind == "weights":                        # a heavy tail, some positions that never got any
        x = np.where(x < 0.1, 0.0, x ** 8)
    elif kind == "ties":                         # few distinct values, both zeros among them
        x = rng.choice([0.0, -0.0, 0.25, 1.5, 3.0], size=shape)
    elif kind == "odd":                          # what no weight is: negatives, infinities, NaN
        x = rng.choice([-1.0, -np.inf, np.inf, np.nan, 0.0, 1e-42, -1e-42, 2.0], size=shape)
    elif kind == "equal":
        x = np.full(shape, 0.125)
    return x.astype(np.float32)


def _case(name, lens, budget, n_sink, n_recent, store, kind="weights", to_other=False, act=None, seed=0, geo=None):
    rng = np.random.default_rng(seed + 7 * budget + len(lens))
    n_seq = len(lens)
    cap = max(max(lens), budget) + 2
    cap += -cap % 128
    parts = (2 if to_other else 1) * n_seq + 1
    g = R.geom(name, slot_ctx=cap, n_slots=parts, **(geo or {}))
    e = R.engine(g)
    perm = rng.permutation(parts)
    src, dst = perm[:n_seq], perm[n_seq:2 * n_seq] if to_other else perm[:n_seq]
    score = _scores(kind, rng, (parts, g.n_kv, cap))
    kept0, pos0 = np.full((n_seq, g.n_kv, budget), -9, dtype=np.int32), np.full(n_seq, -9, dtype=np.int32)
    if store == "slots":
        shape = (parts, g.n_kv, cap, g.rec)
        page = None
    else:
        per = cap // 128
        page = rng.permutation(parts * per).reshape(parts, per).astype(np.int32)
        shape = (parts * per, g.n_kv, 128, g.rec)
    cache = [rng.integers(0, 256, shape, dtype=np.uint8) for _ in range(2)]

    def view(x, s):                              # records [kv head][cap][record] of a partition, as a copy
        return x[s] if page is None else x[page[s]].transpose(1, 0, 2, 3).reshape(g.n_kv, cap, g.rec)

    def store_back(x, s, val):
        if page is None:
            x[s] = val
        else:
            x[page[s]] = val.reshape(g.n_kv, -1, 128, g.rec).transpose(1, 0, 2, 3)

    want_c, want_s = [x.copy() for x in cache], score.copy()
    want_k, want_p = kept0.copy(), pos0.copy()
    for i, n in enumerate(lens):
        if act is not None and not act[i]:
            continue
        m = min(n, budget)
        want_p[i], want_k[i, :, m:] = m, -1
        idx = np.stack([R.evict_list(score[src[i], h, :n], budget, n_sink, n_recent) for h in range(g.n_kv)])
        want_k[i, :, :m] = idx
        h = np.arange(g.n_kv)[:, None]
        want_s[dst[i], :, :m] = score[src[i]][h, idx]
        for t in range(2):
            val = view(want_c[t], dst[i]).copy()
            val[:, :m] = view(cache[t], src[i])[h, idx]
            store_back(want_c[t], dst[i], val)

    dev = [torch.from_numpy(x.reshape(-1)).to(e.device) for x in cache]
    sc, kept = torch.from_numpy(score).to(e.device), torch.from_numpy(kept0).to(e.device)
    pos, pos_out = R.ids(lens, e), torch.from_numpy(pos0).to(e.device)
    kw = dict(n_sink=n_sink, n_recent=n_recent, act=None if act is None else R.ids(act, e))
    part = e.alloc_evict_part(n_seq)
    if store == "slots":
        e.evict(*dev, sc, kept, pos_out, pos, part, budget, kslot=R.ids(src, e),
                kslot_dst=R.ids(dst, e) if to_other else None, **kw)
    else:
        from bruce_engine_b200 import capi
        tab = torch.from_numpy(page).to(e.device)
        desc = capi.CPages(dev[0].data_ptr(), dev[1].data_ptr(), tab.data_ptr(), shape[0], parts, page.shape[1], 128)
        e.evict_paged(desc, sc, kept, pos_out, pos, part, budget, ktab=R.ids(src, e),
                      ktab_dst=R.ids(dst, e) if to_other else None, **kw)
    torch.cuda.synchronize()
    assert e.device_status() == 0
    np.testing.assert_array_equal(kept.cpu().numpy(), want_k)
    np.testing.assert_array_equal(pos_out.cpu().numpy(), want_p)
    np.testing.assert_array_equal(sc.cpu().numpy().view(np.uint32), want_s.view(np.uint32))
    for t in range(2):
        assert (dev[t].cpu().numpy().reshape(shape) == want_c[t]).all(), "KV"[t]


@pytest.mark.parametrize("store", ["slots", "paged"])
@pytest.mark.parametrize("to_other", [False, True])
@pytest.mark.parametrize("name", ["B", "R"])
def test_lists_records_and_scores(name, to_other, store):
    for lens, budget, n_sink, n_recent in (([1], 1, 0, 0), ([2], 1, 0, 0), ([5, 1, 9], 4, 1, 2), ([700, 64, 63, 65], 64, 4, 16),
                                           ([1300, 900], 640, 0, 0), ([4160], 4096, 4, 512), ([3000], 17, 5, 7)):
        _case(name, lens, budget, n_sink, n_recent, store, to_other=to_other, seed=len(lens))


@pytest.mark.parametrize("kind", ["ties", "odd", "equal"])
def test_ties_go_to_the_lower_position_and_nan_goes_first(kind):
    for budget, n_sink, n_recent in ((100, 0, 0), (333, 4, 50), (1999, 1, 1)):
        _case("B", [2000, 1024, 150], budget, n_sink, n_recent, "slots", kind)


def test_edges_of_the_kept_ranges():
    for budget, n_sink, n_recent in ((64, 64, 0), (64, 0, 64), (64, 30, 34), (64, 0, 0), (1, 1, 0), (1, 0, 1), (500, 4, 496)):
        _case("B", [500, 501, 700], budget, n_sink, n_recent, "slots", to_other=bool(budget & 1))


def test_batches():
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(0, 900, 40)]
    _case("B", lens, 256, 4, 32, "slots", act=[int(x) for x in rng.integers(0, 2, 40)])
    _case("R", lens, 256, 4, 32, "paged", to_other=True, act=[int(x) for x in rng.integers(0, 2, 40)])


def test_more_candidates_than_shared_memory_holds():
    for kind in ("weights", "ties"):
        _case("B", [345003], 9001, 4, 100, "slots", kind, to_other=True, geo=dict(n_head=1, n_kv=1))
    _case("B", [345003], 300000, 4, 100, "slots", geo=dict(n_head=1, n_kv=1))


def test_single_sequence_form_and_repeated_trims():
    """One slot's base pointers; the counts go back into pos, so that a captured trim replays while the cache grows."""
    g = R.geom("B", slot_ctx=1024, n_slots=1)
    e = R.engine(g)
    rng = np.random.default_rng(5)
    budget, n_sink, n_recent = 500, 4, 60
    cache = [rng.integers(0, 256, (g.n_kv, 1024, g.rec), dtype=np.uint8) for _ in range(2)]
    score = rng.random((g.n_kv, 1024), dtype=np.float32) ** 8
    dev = [torch.from_numpy(x.copy().reshape(-1)).to(e.device) for x in cache]
    sc, pos = torch.from_numpy(score.copy()).to(e.device), R.ids([900], e)
    kept, part = torch.zeros(1, g.n_kv, budget, dtype=torch.int32, device=e.device), e.alloc_evict_part(1)

    def trim():
        e.evict(*dev, sc, kept, pos, pos, part, budget, n_sink=n_sink, n_recent=n_recent)

    side = torch.cuda.Stream()
    graph = None
    n = 900
    for t in range(4):
        idx = np.stack([R.evict_list(score[h, :n], budget, n_sink, n_recent) for h in range(g.n_kv)])
        m = idx.shape[1]
        h = np.arange(g.n_kv)[:, None]
        score[:, :m] = score[h, idx]
        for x in cache:
            x[:, :m] = x[h, idx]
        if t == 0:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                trim()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                trim()
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert int(pos[0]) == m and (kept.cpu().numpy()[0, :, :m] == idx).all()
        np.testing.assert_array_equal(sc.cpu().numpy(), score)
        for t2 in range(2):
            assert (dev[t2].cpu().numpy().reshape(cache[t2].shape) == cache[t2]).all()
        n = m + (64, 1, 0, 300)[t]
        pos.fill_(n)
    assert e.device_status() == 0


def test_bad_positions_slots_and_clashes_set_the_status_bit():
    g = R.geom("B", slot_ctx=256, n_slots=4)
    e = R.engine(g)
    part = e.alloc_evict_part(2)

    def run(pos, src, dst=None, act=None):
        k, v = e.alloc_kv_layer(False, fill=3)
        score = torch.rand(4, g.n_kv, 256, device=e.device)
        before = score.clone()
        kept = torch.full((len(pos), g.n_kv, 32), -9, dtype=torch.int32, device=e.device)
        out = torch.full((len(pos),), -9, dtype=torch.int32, device=e.device)
        e.evict(k, v, score, kept, out, R.ids(pos, e), part, 32, kslot=R.ids(src, e),
                kslot_dst=None if dst is None else R.ids(dst, e), act=None if act is None else R.ids(act, e))
        torch.cuda.synchronize()
        return e.device_status(), out.tolist(), bool((score == before).all())

    for pos, src, dst in (([257], [0], None), ([-1], [0], None), ([100], [4], None), ([100], [-1], None), ([100], [0], [4]),
                          ([100], [0], [-2])):
        assert run(pos, src, dst) == (1, [-9], True), (pos, src, dst)
    # both write partition 2; one writes what the other reads; the same sequence twice in place
    assert run([100, 100], [0, 1], [2, 2]) == (1, [-9, -9], True)
    st, out, _ = run([100, 100], [0, 1], [1, 2])
    assert st == 1 and out == [-9, 32]
    assert run([100, 100], [1, 1]) == (1, [-9, -9], True)
    # an idle sequence clashes with nobody
    assert run([100, 100], [0, 1], [2, 2], act=[1, 0])[:2] == (0, [32, -9])
    # two targets may share a source
    assert run([100, 100], [0, 0], [2, 3])[:2] == (0, [32, 32])


def test_an_unmapped_page_skips_the_sequence():
    """A hole among the source's or the target's pages sets the status bit; the sequence, and page 0, stay as they are."""
    from bruce_engine_b200 import capi
    g = R.geom("B", slot_ctx=512, n_slots=1)
    e = R.engine(g)
    part = e.alloc_evict_part(2)
    for hole, ok in (((0, 1), False), ((0, 2), True), ((2, 0), False), ((2, 1), True), (None, True)):
        table = np.arange(16, dtype=np.int32).reshape(4, 4)
        if hole:
            table[hole] = (-1, 16)[hole[1] & 1]
        tab = torch.from_numpy(table).to(e.device)
        pool = [torch.randint(0, 256, (16 * g.n_kv * 128 * g.rec,), dtype=torch.uint8, device=e.device) for _ in range(2)]
        before = [x.clone() for x in pool]
        desc = capi.CPages(pool[0].data_ptr(), pool[1].data_ptr(), tab.data_ptr(), 16, 4, 4, 128)
        score = torch.rand(4, g.n_kv, 512, device=e.device)
        kept = torch.full((2, g.n_kv, 100), -9, dtype=torch.int32, device=e.device)
        out = R.ids([-9, -9], e)
        # sequence 0 holds pages 0 and 1 of its row and fills one page of row 2; sequence 1 is sound
        e.evict_paged(desc, score, kept, out, R.ids([200, 130], e), part, 100, ktab=R.ids([0, 1], e), ktab_dst=R.ids([2, 3], e))
        torch.cuda.synchronize()
        assert e.device_status() == (0 if ok else 1) and out.tolist() == [100 if ok else -9, 100], hole
        for a, b in zip(pool, before):
            a, b = a.reshape(16, -1), b.reshape(16, -1)
            assert torch.equal(a[:8], b[:8]) and torch.equal(a[8], b[8]) == (not ok) and not torch.equal(a[12], b[12])


def test_refusals():
    from bruce_engine_b200 import capi
    g = R.geom("B", slot_ctx=256, n_slots=2)
    e = R.engine(g)
    k, v = e.alloc_kv_layer(False, fill=0)
    score, pos = torch.zeros(2, g.n_kv, 256, device=e.device), R.ids([100], e)
    kept, out, part = torch.zeros(1, g.n_kv, 256, dtype=torch.int32, device=e.device), R.ids([0], e), e.alloc_evict_part(1)

    def call(budget=64, n_sink=0, n_recent=0, kslot=R.ids([0], e), **kw):
        e.evict(k, v, kw.pop("score", score), kw.pop("kept", kept), out, pos, part, budget, n_sink, n_recent, kslot=kslot, **kw)

    call()
    for code, kw in ((capi.ERR_ARG, dict(budget=0)), (capi.ERR_ARG, dict(budget=-1)), (capi.ERR_CAPACITY, dict(budget=257, kept=torch.zeros(
                        1, g.n_kv, 257, dtype=torch.int32, device=e.device))),
                     (capi.ERR_ARG, dict(n_sink=-1)), (capi.ERR_ARG, dict(n_recent=-1)), (capi.ERR_ARG, dict(n_sink=40, n_recent=25)),
                     (capi.ERR_ARG, dict(n_sink=65)), (capi.ERR_ARG, dict(n_sink=64, n_recent=2**31 - 1)),
                     (capi.ERR_ARG, dict(kslot=None, kslot_dst=R.ids([1], e)))):
        with pytest.raises(capi.BattnError) as err:
            call(**kw)
        assert err.value.code == code, kw
    for kw in (dict(kept=kept[:, :, :63].contiguous()), dict(score=score[:1].contiguous()), dict(score=score.half()),
               dict(score=score.transpose(1, 2))):
        with pytest.raises(ValueError):
            call(**kw)
    torch.cuda.synchronize()
    assert e.device_status() == 0
