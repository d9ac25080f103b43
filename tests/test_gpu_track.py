"""Attention that accumulates its weights, through the C ABI, against the definition in 64 bits; and the bounded cache it
serves: prompt, decode and eviction together.  Tolerances: bounded_ref.assert_attention, assert_scores."""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R
from tests.gpu_util import dev_q, new_out, to_np

pytestmark = pytest.mark.gpu


def _case(name, lens, rows, store, seed, how="add", act=None):
    """how: "add" (score_in beside score_out), "same" (one buffer), "none" (score_in None)."""
    n_seq = len(lens)
    cap = max(lens) + rows + 2
    cap += -cap % 128
    slots = n_seq + 2
    g = R.geom(name, slot_ctx=cap, n_slots=slots)
    e = R.engine(g)
    rng = np.random.default_rng(seed)
    order = rng.permutation(slots)[:n_seq]
    q, recs = [], []
    for i, p in enumerate(lens):
        qq, k, v = R.draw(g, p + rows, rows, seed * 50 + i)
        q.append(qq)
        recs.append(R.quantised(g, k, v))
    # scores of positions that are not held yet, the call's own included, are NaN: they must not be read
    first = np.full((slots, g.n_kv, cap), np.nan, dtype=np.float32)
    for i, p in enumerate(lens):
        first[order[i], :, :p] = 4 * rng.random((g.n_kv, p)) ** 8
    sin = torch.from_numpy(first).to(e.device)
    sout = sin if how == "same" else torch.full_like(sin, -3.0)
    qd, out = dev_q(e, np.stack(q)), new_out(e, n_seq, rows, g.n_head, g.head_dim)
    pos, part = R.ids(lens, e), e.alloc_track_part(n_seq, rows, sum(lens) + n_seq * rows)
    a = None if act is None else R.ids(act, e)
    given = None if how == "none" else sin
    if store == "paged":
        pg = R.Paged(e, recs, 0, 128, seed)
        tab = torch.full((slots, cap // 128), -1, dtype=torch.int32, device=e.device)
        tab[torch.from_numpy(order.copy()).long(), :pg.table.shape[1]] = pg.table
        pg.desc.table, pg.desc.n_tables, pg.desc.max_pages = tab.data_ptr(), slots, cap // 128
        e.attn_track_paged(out, sout, given, qd, pg.desc, pos, part, rows=rows, ktab=R.ids(order, e), act=a)
    else:
        kvk, kvv = e.alloc_kv_layer(False, fill=0x7F)
        for buf, t in ((kvk, 0), (kvv, 1)):
            R.put(e, buf, {int(s): recs[i] for i, s in enumerate(order)}, False, t)
        e.attn_track(out, sout, given, qd, kvk, kvv, pos, part, rows=rows, kslot=R.ids(order, e), act=a)
    torch.cuda.synchronize()
    assert e.device_status() == 0
    got, sc = to_np(out), sout.cpu().numpy()
    rest = np.ones((slots, cap), dtype=bool)
    for i, p in enumerate(lens):
        what = f"track {name} {store} rows {rows} at {p}"
        if act is not None and not act[i]:
            assert np.isnan(got[i]).all(), what
            continue
        rest[order[i], :p + rows] = False
        R.assert_attention(got[i], R.attend64(g, q[i], *recs[i], p), g, recs[i][1], what)
        want = R.score64(g, q[i], recs[i][0], p, None if how == "none" else first[order[i]])
        R.assert_scores(sc[order[i], :, :p + rows], want, g, q[i], recs[i][0], p, what)
    kept = (first if how == "same" else np.full_like(first, -3.0)).transpose(0, 2, 1)[rest]
    np.testing.assert_array_equal(sc.transpose(0, 2, 1)[rest], kept)      # everything else is as it was


@pytest.mark.parametrize("store", ["slots", "paged"])
@pytest.mark.parametrize("name", ["B", "B32", "R", "B1", "B8"])
@pytest.mark.parametrize("how", ["add", "same", "none"])
def test_one_token_of_many_sequences(name, store, how):
    _case(name, [0, 1, 62, 63, 64, 127, 500, 2047, 2048, 3001], 1, store, 3, how)


@pytest.mark.parametrize("name", ["B", "R"])
def test_one_token_of_one_sequence(name):
    for p in (0, 5, 64, 9000, 40001):
        _case(name, [p], 1, "slots", p + 1, "same")


@pytest.mark.parametrize("store", ["slots", "paged"])
@pytest.mark.parametrize("name,rows", [("B", 2), ("B", 7), ("B", 33), ("B32", 100), ("B", 512), ("R", 3), ("R", 32), ("R", 201),
                                       ("B8", 50), ("B1", 129)])
def test_prompt_chunk(name, rows, store):
    for p, how in ((0, "none"), (1, "add"), (127, "same"), (1700, "same"), (2001, "none")):
        _case(name, [p], rows, store, rows + p, how)


def test_a_long_prompt():
    _case("B", [16000], 384, "slots", 1, "same")
    _case("R16", [16000], 40, "paged", 1, "none")


def test_idle_sequences_are_left_alone():
    _case("B", [500, 40, 300, 9], 1, "slots", 5, "same", act=[1, 0, 1, 0])
    _case("B", [500], 1, "slots", 5, "same", act=[0])
    for name in ("B", "R"):
        for rows in (2, 100):
            _case(name, [600], rows, "paged", 6, "same", act=[0])
            # what an idle sequence's position and slot hold does not matter
            g = R.geom(name, slot_ctx=512)
            e = R.engine(g)
            q = torch.zeros(1, rows, g.n_head, g.head_dim, dtype=e.q_torch, device=e.device)
            out, score = new_out(e, 1, rows, g.n_head, g.head_dim), torch.ones(1, g.n_kv, 512, device=e.device)
            for early in (False, True):
                e.set_early_kv_stream(early)
                e.attn_track(out, score, score, q, *e.alloc_kv_layer(False, fill=0), R.ids([-7], e), e.alloc_track_part(1, rows, 512),
                             rows=rows, kslot=R.ids([99], e), act=R.ids([0], e))
                torch.cuda.synchronize()
                assert e.device_status() == 0 and torch.isnan(out).all() and (score == 1).all()


def test_attention_output_is_the_plain_calls():
    """What the call adds does not change what it computes: the decode output is battn_decode's, bit for bit."""
    g = R.geom("B", slot_ctx=4096)
    e = R.engine(g)
    for p in (0, 77, 4000):
        q, k, v = R.draw(g, p + 1, 1, p)
        recs = R.quantised(g, k, v)
        kvk, kvv = e.alloc_kv_layer(False, fill=0x7F)
        R.put(e, kvk, {0: recs}, False, 0)
        R.put(e, kvv, {0: recs}, False, 1)
        a, b = new_out(e, 1, 1, g.n_head, g.head_dim), new_out(e, 1, 1, g.n_head, g.head_dim)
        qd, pos = dev_q(e, q[None]), R.ids([p], e)
        e.launch_attn_m(a, qd, kvk, kvv, pos, e.alloc_part(1, 1), 1)
        s = torch.zeros(g.n_kv, 4096, device=e.device)
        e.attn_track(b, s, s, qd, kvk, kvv, pos, e.alloc_track_part(1, 1, p + 1))
        torch.cuda.synchronize()
        assert torch.equal(a, b)


def test_two_graphs_share_a_workspace_and_repeat():
    """Two captured calls on one workspace, replayed in turn: the same bits every time."""
    g = R.geom("B", slot_ctx=2048, n_slots=3)
    e = R.engine(g)
    lens = [1500, 3, 800]
    kvk, kvv = (torch.randint(0, 60, (e.kv_layer_bytes(False),), dtype=torch.uint8, device=e.device) for _ in range(2))
    pos, slots, part = R.ids(lens, e), R.ids([0, 1, 2], e), e.alloc_track_part(3, 100, 4000)
    q1 = torch.randn(3, 1, g.n_head, g.head_dim, device=e.device).half()
    q2 = torch.randn(1, 100, g.n_head, g.head_dim, device=e.device).half()
    o1, o2 = torch.empty_like(q1), torch.empty_like(q2)
    s1, s2 = (torch.zeros(3, g.n_kv, 2048, device=e.device) for _ in range(2))

    def one():
        e.attn_track(o1, s1, None, q1, kvk, kvv, pos, part, kslot=slots)

    def two():
        e.attn_track(o2, s2, None, q2, kvk, kvv, pos[2:], part, rows=100, kslot=slots[2:])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(); two()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    first = [t.clone() for t in (o1, s1, o2, s2)]
    graphs = []
    for f in (one, two):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f()
        graphs.append(gr)
    for _ in range(20):
        for t in (o1, s1, o2, s2):
            t.fill_(7)
        graphs[0].replay(); graphs[1].replay()
        torch.cuda.synchronize()
        for got, want, clean in ((o1, first[0], None), (o2, first[2], None), (s1, first[1], lens), (s2, first[3], [0, 0, 900])):
            if clean is None:
                assert torch.equal(got, want)
            else:
                for i, n in enumerate(clean):
                    assert torch.equal(got[i, :, :n], want[i, :, :n])
    assert e.device_status() == 0


def test_offsets_past_32_bits():
    """The last slot of a 5.7 GB cache (and of pages as far) gives what slot 0 gives: weights, sinks and eviction."""
    from bruce_engine_b200 import capi
    g = R.geom("B", slot_ctx=262144, n_slots=20, window=128)
    e = R.engine(g)
    kvk, kvv = (e.alloc_kv_layer(False)[0] for _ in range(2))
    assert kvk.numel() > 2 ** 32
    for rows in (1, 40):
        q, k, v = R.draw(g, 500 + rows, rows, rows)
        recs = R.quantised(g, k, v)
        for buf, r in ((kvk, recs[0]), (kvv, recs[1])):
            for s in (0, 19):
                buf.view(20, g.n_kv, -1, g.rec)[s, :, :500 + rows].copy_(torch.from_numpy(r.copy()))
        qd, pos = dev_q(e, q[None]), R.ids([500], e)
        score = torch.zeros(20, g.n_kv, g.slot_ctx, device=e.device)
        res = {}
        # pages of 128: the whole cache seen as a pool, page p of the row at the pool's end or start
        n_pages = kvk.numel() // (g.n_kv * 128 * g.rec)
        for s in (0, 19):
            out, out2 = new_out(e, 1, rows, g.n_head, g.head_dim), new_out(e, 1, rows, g.n_head, g.head_dim)
            kept, left = torch.zeros(1, g.n_kv, 200, dtype=torch.int32, device=e.device), R.ids([0], e)
            slot = R.ids([s], e)
            e.attn_track(out, score, score, qd, kvk, kvv, pos, e.alloc_track_part(1, rows, 600), rows=rows, kslot=slot)
            e.attn_sinks(out2, qd, kvk, kvv, e.sinks(4), pos, e.alloc_part(1, rows), rows=rows, kslot=slot, is_swa=False)
            e.evict(kvk, kvv, score, kept, left, pos, e.alloc_evict_part(1), 200, n_recent=50, kslot=slot)
            res[s] = [out, out2, kept, left, score[s, :, :200].clone(),
                      kvk.view(20, g.n_kv, -1, g.rec)[s, :, :200].clone(), kvv.view(20, g.n_kv, -1, g.rec)[s, :, :200].clone()]
        for s, first in ((0, 0), (19, n_pages - 6)):
            tab = torch.arange(first, first + 5, dtype=torch.int32, device=e.device)[None].contiguous()
            for buf, r in ((kvk, recs[0]), (kvv, recs[1])):
                pool = buf[:n_pages * g.n_kv * 128 * g.rec].view(n_pages, g.n_kv, 128, g.rec)
                for p in range(5):
                    x = torch.from_numpy(r[:, 128 * p:128 * (p + 1)].copy())
                    pool[first + p, :, :x.shape[1]].copy_(x)
            desc = capi.CPages(kvk.data_ptr(), kvv.data_ptr(), tab.data_ptr(), n_pages, 1, 5, 128)
            out, sc = new_out(e, 1, rows, g.n_head, g.head_dim), torch.zeros(1, g.n_kv, 640, device=e.device)
            e.attn_track_paged(out, sc, None, qd, desc, pos, e.alloc_track_part(1, rows, 600), rows=rows)
            res[s] += [out, sc]
        torch.cuda.synchronize()
        assert e.device_status() == 0
        for a, b in zip(res[0], res[19]):
            assert torch.equal(a, b)
        R.assert_attention(to_np(res[19][0])[0], R.attend64(g, q, *recs, 500), g, recs[1], "far slot")
        assert torch.equal(res[19][0], res[19][7])


def test_a_first_call_may_be_captured():
    """In a fresh process every new call is captured before it ever ran, then replayed."""
    import os
    import subprocess
    import sys
    code = """
import torch
from tests import bounded_ref as R
for name in ("B", "R16"):
    g = R.geom(name, window=128, slot_ctx=2048, n_slots=20)
    e = R.engine(g)
    kv = [torch.randint(0, 60, (e.kv_layer_bytes(False),), dtype=torch.uint8, device="cuda") for _ in range(2)]
    ring = e.alloc_kv_layer(True, fill=0)
    sk, bk, bv = e.alloc_sinks(4)
    q = {r: torch.randn(r, g.n_head, g.head_dim, device="cuda").half() for r in (1, 8, 20, 90)}
    o = {r: torch.zeros_like(x) for r, x in q.items()}
    s = torch.zeros(20, g.n_kv, 2048, device="cuda")
    pos, ks = R.ids([900] * 20, e), R.ids(range(20), e)
    part, tp, ep = e.alloc_part(20, 90), e.alloc_track_part(20, 90, 40000), e.alloc_evict_part(20)
    kept, left = torch.zeros(20, g.n_kv, 300, dtype=torch.int32, device="cuda"), R.ids([0] * 20, e)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        e.sinks_store(*ring, sk, pos[:1], kslot=ks[:1])
        for r in (1, 8, 90):
            e.attn_sinks(o[r], q[r], *kv, e.sinks(4), pos[:1], part, rows=r, kslot=ks[:1], is_swa=False)
        e.attn_sinks(o[20], q[20], *kv, e.sinks(4), pos, part, kslot=ks, is_swa=False)
        e.attn_track(o[1], s, s, q[1], *kv, pos[:1], tp, kslot=ks[:1])
        e.attn_track(o[20], s, s, q[20], *kv, pos, tp, kslot=ks)
        e.attn_track(o[90], s, s, q[90], *kv, pos[:1], tp, rows=90, kslot=ks[:1])
        e.evict(*kv, s, kept, left, pos, ep, 300, kslot=ks)
    graph.replay()
    torch.cuda.synchronize()
    assert e.device_status() == 0 and left.tolist() == [300] * 20 and all(torch.isfinite(x).all() for x in o.values())
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_calls_on_two_streams_at_once():
    """Two streams, each with its own buffers and scratch, on one handle: what each computes alone."""
    g = R.geom("B", slot_ctx=8192, n_slots=2)
    e = R.engine(g)

    def job(seed):
        torch.manual_seed(seed)
        kv = [torch.randint(0, 60, (e.kv_layer_bytes(False),), dtype=torch.uint8, device=e.device) for _ in range(2)]
        q1 = torch.randn(2, 1, g.n_head, g.head_dim, device=e.device).half()
        q2 = torch.randn(1, 200, g.n_head, g.head_dim, device=e.device).half()
        o1, o2, s = torch.empty_like(q1), torch.empty_like(q2), torch.zeros(2, g.n_kv, 8192, device=e.device)
        part, ep = e.alloc_track_part(2, 200, 16384), e.alloc_evict_part(2)
        kept, left = torch.zeros(2, g.n_kv, 3000, dtype=torch.int32, device=e.device), R.ids([0, 0], e)
        pos, ks = R.ids([7000, 6000], e), R.ids([0, 1], e)

        def run():
            e.attn_track(o1, s, s, q1, *kv, pos, part, kslot=ks)
            e.attn_track(o2, s, s, q2, *kv, pos[1:], part, rows=200, kslot=ks[1:])
            e.evict(*kv, s, kept, left, pos, ep, 3000, n_sink=4, n_recent=100, kslot=ks)
            e.attn_track(o1, s, s, q1, *kv, left, part, kslot=ks)
        return run, [o1, o2, s, kept, left] + kv

    alone = []
    for seed in (1, 2):
        run, got = job(seed)
        run()
        torch.cuda.synchronize()
        alone.append([t.clone() for t in got])
    for _ in range(3):
        jobs = [job(seed) for seed in (1, 2)]
        streams = [torch.cuda.Stream() for _ in jobs]
        torch.cuda.synchronize()
        for (run, _), st in zip(jobs, streams):
            with torch.cuda.stream(st):
                run()
        torch.cuda.synchronize()
        assert e.device_status() == 0
        for (_, got), want in zip(jobs, alone):
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_a_slot_named_twice():
    """Two active sequences on one slot: both outputs, the status bit, and the slot's scores as they were; the same slot
    twice is fine when one of the two is idle, and for the others nothing changes."""
    g = R.geom("B", slot_ctx=512, n_slots=4)
    e = R.engine(g)
    kvk, kvv = (torch.randint(0, 60, (e.kv_layer_bytes(False),), dtype=torch.uint8, device=e.device) for _ in range(2))
    q = torch.randn(3, 1, g.n_head, g.head_dim, device=e.device).half()
    pos, part = R.ids([300, 200, 100], e), e.alloc_track_part(3, 1, 700)
    ref, o_ref = torch.full((4, g.n_kv, 512), 5.0, device=e.device), torch.empty_like(q)
    e.attn_track(o_ref, ref, None, q, kvk, kvv, pos, part, kslot=R.ids([0, 1, 2], e))
    for slots, act, status in (([1, 1, 2], [1, 1, 1], 1), ([1, 1, 2], [0, 1, 1], 0)):
        score, o = torch.full_like(ref, 5.0), torch.full_like(q, 9.0)
        e.attn_track(o, score, None, q, kvk, kvv, pos, part, kslot=R.ids(slots, e), act=R.ids(act, e))
        torch.cuda.synchronize()
        assert e.device_status() == status
        assert torch.equal(o[1:], o_ref[1:]) and torch.equal(score[2], ref[2]) and (score[0] == 5.0).all()
        assert (score[1] == 5.0).all() if status else torch.equal(score[1], ref[1])


def test_the_largest_batch():
    """1024 sequences of a few positions, ragged, some idle: tracked, attended with sinks, evicted."""
    g = R.geom("B", slot_ctx=128, n_slots=1024, window=64)
    e = R.engine(g)
    rng = np.random.default_rng(8)
    lens = rng.integers(0, 120, 1024)
    act = (rng.random(1024) < 0.9).astype(np.int32)
    q, k, v = R.draw(g, 128, 1, 4)
    recs = R.quantised(g, k, v)
    kvk, kvv = e.alloc_kv_layer(False, fill=0)
    for buf, r in ((kvk, recs[0]), (kvv, recs[1])):
        buf.copy_(torch.from_numpy(np.broadcast_to(r[None, :, :128], (1024,) + r[:, :128].shape).reshape(-1).copy()))
    qd = dev_q(e, np.broadcast_to(q[None], (1024,) + q.shape))
    order = rng.permutation(1024)
    pos, ks, a = R.ids(lens, e), R.ids(order, e), R.ids(act, e)
    score = torch.full((1024, g.n_kv, 128), float("nan"), device=e.device)
    out, out2 = new_out(e, 1024, 1, g.n_head, g.head_dim), new_out(e, 1024, 1, g.n_head, g.head_dim)
    e.attn_track(out, score, None, qd, kvk, kvv, pos, e.alloc_track_part(1024, 1, int(lens.sum()) + 1024), kslot=ks, act=a)
    e.attn_sinks(out2, qd, kvk, kvv, e.sinks(4), pos, e.alloc_part(1024, 1), kslot=ks, act=a, is_swa=False)
    kept, left = torch.full((1024, g.n_kv, 40), -9, dtype=torch.int32, device=e.device), R.ids([-9] * 1024, e)
    torch.cuda.synchronize()
    sc = score.cpu().numpy()
    e.evict(kvk, kvv, score, kept, left, pos, e.alloc_evict_part(1024), 40, n_sink=2, n_recent=8, kslot=ks, act=a)
    torch.cuda.synchronize()
    assert e.device_status() == 0
    got, got2, kept, left = to_np(out), to_np(out2), kept.cpu().numpy(), left.cpu().numpy()
    for i in range(0, 1024, 7):
        p = int(lens[i])
        if not act[i]:
            assert np.isnan(got[i]).all() and np.isnan(got2[i]).all() and left[i] == -9 and (kept[i] == -9).all()
            continue
        R.assert_attention(got[i], R.attend64(g, q, *recs, p), g, recs[1], f"track {i}")
        R.assert_attention(got2[i], R.attend64(g, q, *recs, p, 4, 64), g, recs[1], f"sinks {i}")
        want = R.score64(g, q, recs[0], p, None)
        R.assert_scores(sc[order[i], :, :p + 1], want, g, q, recs[0], p, f"scores {i}")
        assert left[i] == min(p, 40)
        for h in range(g.n_kv):
            idx = R.evict_list(sc[order[i], h, :p], 40, 2, 8)
            assert (kept[i, h, :len(idx)] == idx).all() and (kept[i, h, len(idx):] == -1).all()


def test_a_workspace_that_is_too_small_for_the_positions():
    g = R.geom("B", slot_ctx=4096, n_slots=2)
    e = R.engine(g)
    kvk, kvv = e.alloc_kv_layer(False, fill=0)
    q = torch.zeros(2, 1, g.n_head, g.head_dim, dtype=torch.float16, device=e.device)
    part = e.alloc_track_part(2, 1, 2000)
    score = torch.full((2, g.n_kv, 4096), 5.0, device=e.device)
    for lens, status in (([1000, 900], 0), ([4000, 10], 4), ([1, 1], 0)):
        out = new_out(e, 2, 1, g.n_head, g.head_dim)
        score.fill_(5.0)
        e.attn_track(out, score, score, q, kvk, kvv, R.ids(lens, e), part, kslot=R.ids([0, 1], e))
        torch.cuda.synchronize()
        assert e.device_status() == status
        assert bool(torch.isnan(out).all()) == bool(status) and bool((score == 5.0).all()) == bool(status)


def test_bad_positions_and_slots_set_the_status_bit():
    g = R.geom("B", slot_ctx=512, n_slots=2)
    e = R.engine(g)
    kvk, kvv = e.alloc_kv_layer(False, fill=0)
    part = e.alloc_track_part(1, 100, 600)
    for rows in (1, 4, 100):
        for p, s in ((-1, 0), (513 - rows, 0), (5, 2), (5, -1)):
            out = new_out(e, 1, rows, g.n_head, g.head_dim)
            score = torch.full((2, g.n_kv, 512), 5.0, device=e.device)
            q = torch.zeros(1, rows, g.n_head, g.head_dim, dtype=torch.float16, device=e.device)
            e.attn_track(out, score, score, q, kvk, kvv, R.ids([p], e), part, rows=rows, kslot=R.ids([s], e))
            torch.cuda.synchronize()
            assert e.device_status() == 1 and torch.isnan(out).all() and (score == 5.0).all(), (rows, p, s)


def test_refusals():
    from bruce_engine_b200 import capi
    g = R.geom("B", slot_ctx=1024, n_slots=2)
    e = R.engine(g)
    cache = e.alloc_kv_layer(False, fill=0)
    score, part = torch.zeros(2, g.n_kv, 1024, device=e.device), e.alloc_track_part(2, 512, 2048)

    def call(rows=1, n=1, part=part, score=score, into=None, **kw):
        q = torch.zeros(n, rows, g.n_head, g.head_dim, dtype=torch.float16, device=e.device)
        e.attn_track(torch.empty_like(q), score if into is None else into, score, q, *cache, R.ids([5] * n, e), part, rows=rows,
                     kslot=R.ids(range(n), e))

    call()
    for code, kw in ((capi.ERR_CAPACITY, dict(rows=2, n=2)), (capi.ERR_CAPACITY, dict(rows=513)),
                     (capi.ERR_CAPACITY, dict(part=part[:256])), (capi.ERR_CAPACITY, dict(rows=100, part=part[:4096])),
                     (capi.ERR_ARG, dict(part=part[8:])),
                     (capi.ERR_ARG, dict(into=torch.zeros(score.numel() + 1, device=e.device)[1:]))):
        with pytest.raises(capi.BattnError) as err:
            call(**kw)
        assert err.value.code == code, kw
    for kw in (dict(score=score[:1]), dict(score=score.double()), dict(score=score.transpose(1, 2))):
        with pytest.raises(ValueError):
            call(**kw)
    import ctypes
    n = ctypes.c_size_t()
    for args in ((0, 1, 1), (1, 0, 1), (1, 1, -1)):
        assert e.lib.battn_track_workspace_bytes(e.h, *args, n) == capi.ERR_ARG
    torch.cuda.synchronize()
    assert e.device_status() == 0


@pytest.mark.parametrize("name", ["B", "R"])
def test_a_conversation_in_a_bounded_cache(name):
    """A prompt of 300 tokens, cut to 128, then 120 tokens with a trim whenever 160 are held: append, attend and accumulate,
    evict.  Every step is checked against 64 bits, starting from the scores the previous step left."""
    budget, n_sink, n_recent, limit = 128, 4, 32, 160
    g = R.geom(name, slot_ctx=512, n_slots=2)
    e = R.engine(g)
    q, k, v = R.draw(g, 420, 420, 77)
    kvk, kvv = e.alloc_kv_layer(False, fill=0x7F)
    slot, pos = R.ids([1], e), R.ids([0], e)
    score = torch.full((2, g.n_kv, 512), float("nan"), device=e.device)
    kept = torch.zeros(1, g.n_kv, budget, dtype=torch.int32, device=e.device)
    part, epart = e.alloc_track_part(1, 300, 512), e.alloc_evict_part(1)
    krec, vrec = (np.zeros((g.n_kv, 0, g.rec), dtype=np.uint8) for _ in range(2))
    held, at = 0, 0
    while at < 420:
        rows = 300 if at == 0 else 1
        before = score.cpu().numpy()[1]
        kd, vd = (torch.from_numpy(x[at:at + rows]).to(e.device) for x in (k, v))
        qd = torch.from_numpy(q[at:at + rows]).to(e.device).to(e.q_torch)[None].contiguous()
        out = new_out(e, 1, rows, g.n_head, g.head_dim)
        e.qkv_prep_store(kd, vd, kvk, kvv, pos, kslot=slot, rows=rows)
        e.attn_track(out, score, score, qd, kvk, kvv, pos, part, rows=rows, kslot=slot)
        new = R.quantised(g, k[at:at + rows], v[at:at + rows])
        krec, vrec = np.concatenate([krec, new[0]], 1), np.concatenate([vrec, new[1]], 1)
        torch.cuda.synchronize()
        what = f"token {at}"
        R.assert_attention(to_np(out)[0], R.attend64(g, q[at:at + rows], krec, vrec, held), g, vrec, what)
        now = score.cpu().numpy()[1]
        R.assert_scores(now[:, :held + rows], R.score64(g, q[at:at + rows], krec, held, before), g, q[at:at + rows], krec, held, what)
        pos += rows
        held, at = held + rows, at + rows
        if held >= limit:
            e.evict(kvk, kvv, score, kept, pos, pos, epart, budget, n_sink=n_sink, n_recent=n_recent, kslot=slot)
            torch.cuda.synchronize()
            idx = np.stack([R.evict_list(now[h, :held], budget, n_sink, n_recent) for h in range(g.n_kv)])
            np.testing.assert_array_equal(kept.cpu().numpy()[0], idx)
            h = np.arange(g.n_kv)[:, None]
            krec, vrec, held = krec[h, idx], vrec[h, idx], budget
            assert int(pos[0]) == budget
            np.testing.assert_array_equal(score.cpu().numpy()[1, :, :budget], now[h, idx])
            got = kvk.cpu().numpy().reshape(2, g.n_kv, 512, g.rec)[1, :, :budget]
            assert (got == krec).all()
    assert e.device_status() == 0
