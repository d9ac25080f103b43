"""Sliding-window attention with sinks, through the C ABI, against the definition in 64 bits.

Every cached position a row must not see holds NaN scales (0x7F7F) or lies on an unmapped page.  Tolerances:
bounded_ref.assert_attention."""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R
from tests.gpu_util import dev_q, new_out, to_np

pytestmark = pytest.mark.gpu


def _case(name, window, lens, rows, n_sink, store, seed, act=None):
    """One call over len(lens) sequences with `lens` positions before the rows; compares every active sequence."""
    n_seq = len(lens)
    cap = max(lens) + rows + 2
    cap += -cap % 256
    slots = n_seq + 2
    g = R.geom(name, window=window, slot_ctx=cap, n_slots=slots)
    e = R.engine(g)
    order = np.random.default_rng(seed).permutation(slots)[:n_seq]             # partition of each sequence
    q, recs = [], []
    for i, p in enumerate(lens):
        qq, k, v = R.draw(g, p + rows, rows, seed * 50 + i)
        q.append(qq)
        recs.append(R.quantised(g, k, v))
    # poison what no row of the call sees: below the first row's window, past the sinks
    held = []
    for i, p in enumerate(lens):
        kr, vr = (x.copy() for x in recs[i])
        lo = max(0, p + 1 - window)
        kr[:, min(n_sink, lo):lo] = 0x7F
        vr[:, min(n_sink, lo):lo] = 0x7F
        held.append((kr, vr))
    qd = dev_q(e, np.stack(q))
    out = new_out(e, n_seq, rows, g.n_head, g.head_dim)
    pos, part = R.ids(lens, e), e.alloc_part(n_seq, rows)
    a = None if act is None else R.ids(act, e)
    keep = []
    if store == "paged":
        gap = lambda i, p: p * 128 >= n_sink and (p + 1) * 128 <= lens[i] + 1 - window
        pg = R.Paged(e, held, 0, 128, seed, skip=gap)
        tab = torch.full((slots, pg.table.shape[1]), -1, dtype=torch.int32, device=e.device)
        tab[torch.from_numpy(order.copy()).long()] = pg.table
        pg.desc.table, pg.desc.n_tables = tab.data_ptr(), slots
        keep = [tab, pg]
        e.attn_sinks_paged(out, qd, pg.desc, e.sinks(n_sink), pos, part, rows=rows, ktab=R.ids(order, e), act=a)
    else:
        ring = store == "ring"
        kvk, kvv = e.alloc_kv_layer(ring, fill=0x7F)
        R.put(e, kvk, {int(s): held[i] for i, s in enumerate(order)}, ring, 0)
        R.put(e, kvv, {int(s): held[i] for i, s in enumerate(order)}, ring, 1)
        sk = e.sinks(n_sink)
        if ring:
            sk, bk, bv = e.alloc_sinks(n_sink)
            for buf, t in ((bk, 0), (bv, 1)):
                host = np.full((slots, g.n_kv, sk.cap, g.rec), 0x7F, dtype=np.uint8)
                for i, s in enumerate(order):
                    x = held[i][t][:, :sk.cap]
                    host[s][:, :x.shape[1]] = x
                buf.copy_(torch.from_numpy(host.reshape(-1)))
            keep = [bk, bv]
        e.attn_sinks(out, qd, kvk, kvv, sk, pos, part, rows=rows, kslot=R.ids(order, e), act=a, is_swa=ring)
    torch.cuda.synchronize()
    assert e.device_status() == 0
    got = to_np(out)
    for i, p in enumerate(lens):
        if act is not None and not act[i]:
            assert np.isnan(got[i]).all(), "an idle sequence was written"
            continue
        want = R.attend64(g, q[i], *recs[i], p, n_sink, window)
        R.assert_attention(got[i], want, g, recs[i][1], f"sinks {name} {store} rows {rows} at {p}, window {window}, {n_sink} sinks")
    del keep


@pytest.mark.parametrize("store", ["ring", "slots", "paged"])
@pytest.mark.parametrize("name", ["B", "B32", "R"])
@pytest.mark.parametrize("n_sink", [0, 1, 4, 64, 100])
def test_decode(name, store, n_sink):
    # one key, inside the sinks, around the window's first steps, tile borders, and far past both
    _case(name, 128, [0, 3, 63, 127, 128, 129, 191, 255, 300, 1001], 1, n_sink, store, 11 + n_sink)


@pytest.mark.parametrize("store", ["ring", "paged"])
@pytest.mark.parametrize("name,rows", [("B", 2), ("B", 5), ("B", 8), ("R", 3), ("R", 8), ("B1", 8), ("B8", 4), ("B8", 2)])
def test_verify(name, rows, store):
    _case(name, 256, [0, 2, 120, 252, 255, 256, 700], rows, 5, store, 31 + rows)


@pytest.mark.parametrize("store", ["ring", "slots", "paged"])
@pytest.mark.parametrize("name,rows", [("B", 9), ("B", 40), ("B32", 129), ("B", 256), ("R", 9), ("R", 70), ("R", 201), ("B8", 5),
                                       ("B1", 150)])
def test_prompt_chunk(name, rows, store):
    for p, n_sink in ((0, 4), (37, 130), (250, 4), (900, 64), (2001, 0)):
        _case(name, 256, [p], rows, n_sink, store, rows + p)


def test_the_usual_window():
    for name, window in (("B", 4096), ("R16", 1024)):
        for rows, p in ((1, 20000), (8, 9000), (512, 9777)):
            _case(name, window, [p], rows, 4, "ring", rows)


def test_idle_sequences_are_left_alone():
    for rows in (1, 4, 8):
        _case("B", 128, [500, 40, 300], rows, 4, "ring", 5, act=[1, 0, 1])
    for store in ("ring", "paged"):
        _case("B", 128, [600], 100, 4, store, 6, act=[0])
        _case("R", 128, [600], 100, 4, store, 6, act=[0])


def test_no_sinks_equals_the_window_call():
    """On a ring and with n_sink = 0 the call computes what the plain window call does, bit for bit (young sequences
    read their first tile from the sink buffers, which hold the same records)."""
    g = R.geom("B", window=256, slot_ctx=4096)
    e = R.engine(g)
    for p, rows in ((1500, 1), (1500, 4), (1500, 8), (1500, 200)):
        q, k, v = R.draw(g, p + rows, rows, p + rows)
        kr, vr = R.quantised(g, k, v)
        kvk, kvv = e.alloc_kv_layer(True, fill=0x7F)
        R.put(e, kvk, {0: (kr, vr)}, True, 0)
        R.put(e, kvv, {0: (kr, vr)}, True, 1)
        sk, bk, bv = e.alloc_sinks(0)
        qd, pos, part = dev_q(e, q[None]), R.ids([p], e), e.alloc_part(1, rows)
        a, b = new_out(e, 1, rows, g.n_head, g.head_dim), new_out(e, 1, rows, g.n_head, g.head_dim)
        e.launch_attn_m(a, qd, kvk, kvv, pos, part, rows, is_swa=True)
        e.attn_sinks(b, qd, kvk, kvv, sk, pos, part, rows=rows)
        torch.cuda.synchronize()
        assert torch.equal(a, b)


def test_one_slot_of_a_layer():
    """The single-sequence form: slot base pointers of the ring and of the sink buffers give what kslot gives."""
    g = R.geom("B", window=128, slot_ctx=512, n_slots=3)
    e = R.engine(g)
    q, k, v = R.draw(g, 700, 60, 21)
    kr, vr = R.quantised(g, k, v)
    kvk, kvv = e.alloc_kv_layer(True, fill=0x7F)
    R.put(e, kvk, {2: (kr, vr)}, True, 0)
    R.put(e, kvv, {2: (kr, vr)}, True, 1)
    sk, bk, bv = e.alloc_sinks(130)
    for buf, r in ((bk, kr), (bv, vr)):
        buf.view(3, g.n_kv, sk.cap, g.rec)[2].copy_(torch.from_numpy(r[:, :sk.cap].copy()))
    one = e.sinks(100, bk.view(3, -1)[2], bv.view(3, -1)[2], cap=sk.cap)
    sk = e.sinks(100, bk, bv)
    for rows in (1, 8, 60):
        qd, pos, part = dev_q(e, q[None, :rows]), R.ids([700 - rows], e), e.alloc_part(1, rows)
        a, b = new_out(e, 1, rows, g.n_head, g.head_dim), new_out(e, 1, rows, g.n_head, g.head_dim)
        e.attn_sinks(a, qd, kvk, kvv, sk, pos, part, rows=rows, kslot=R.ids([2], e))
        n = kvk.numel() // 3
        e.attn_sinks(b, qd, kvk[2 * n:], kvv[2 * n:], one, pos, part, rows=rows)
        torch.cuda.synchronize()
        assert torch.equal(a, b)
        R.assert_attention(to_np(a)[0], R.attend64(g, q[:rows], kr, vr, 700 - rows, 100, 128), g, vr, f"rows {rows}")


@pytest.mark.parametrize("early", [False, True])
def test_a_stream_from_its_first_token(early):
    """Prompt chunk, then single tokens past two windows: append, keep the sinks, attend, in a captured and replayed step;
    the sinks come out of the ring before it overwrites them."""
    window, n_sink, first, steps, n_seq = 64, 5, 40, 200, 3
    g = R.geom("B", window=window, slot_ctx=512, n_slots=n_seq)
    e = R.engine(g)
    e.set_early_kv_stream(early)
    total = first + steps
    qs, ks, vs, recs = [], [], [], []
    for i in range(n_seq):
        q, k, v = R.draw(g, total, total, 90 + i)
        qs.append(q); ks.append(k); vs.append(v)
        recs.append(R.quantised(g, k, v))
    kvk, kvv = e.alloc_kv_layer(True, fill=0x7F)
    sk, bk, bv = e.alloc_sinks(n_sink)
    slots, pos = R.ids(range(n_seq), e), R.ids([0] * n_seq, e)
    dk, dv = (torch.from_numpy(np.stack(x)).to(e.device) for x in (ks, vs))
    dq = torch.from_numpy(np.stack(qs)).to(e.device).half()
    e.qkv_prep_store(dk[:, :first].contiguous(), dv[:, :first].contiguous(), kvk, kvv, pos, kslot=slots, rows=first, is_swa=True)
    e.sinks_store(kvk, kvv, sk, pos, kslot=slots, rows=first)
    part = e.alloc_part(n_seq, 64)
    out = new_out(e, 1, first, g.n_head, g.head_dim)
    one = R.ids([1], e)
    e.attn_sinks(out, dq[1:2, :first].contiguous(), kvk, kvv, sk, pos[:1], part, rows=first, kslot=one)
    torch.cuda.synchronize()
    R.assert_attention(to_np(out)[0], R.attend64(g, qs[1][:first], *recs[1], 0, n_sink, window), g, recs[1][1], "first chunk")
    pos.fill_(first)
    bufs = {n: torch.empty(n_seq, 1, h, g.head_dim, dtype=t, device=e.device)
            for n, h, t in (("q", g.n_head, torch.float16), ("k", g.n_kv, torch.float32), ("v", g.n_kv, torch.float32))}
    o = new_out(e, n_seq, 1, g.n_head, g.head_dim)

    def step():
        e.qkv_prep_store(bufs["k"], bufs["v"], kvk, kvv, pos, kslot=slots, is_swa=True)
        e.sinks_store(kvk, kvv, sk, pos, kslot=slots)
        e.attn_sinks(o, bufs["q"], kvk, kvv, sk, pos, part, kslot=slots)

    side = torch.cuda.Stream()
    for t in range(steps):
        p = first + t
        bufs["q"].copy_(dq[:, p:p + 1]); bufs["k"].copy_(dk[:, p:p + 1]); bufs["v"].copy_(dv[:, p:p + 1])
        if t == 0:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        else:
            graph.replay()
        if t in (0, 1, 23, 24, 25, 87, 88, 90, 150, steps - 1):
            torch.cuda.synchronize()
            got = to_np(o)
            for i in range(n_seq):
                R.assert_attention(got[i], R.attend64(g, qs[i][p:p + 1], *recs[i], p, n_sink, window), g, recs[i][1],
                                   f"token {p} of {i}")
        pos += 1
    assert e.device_status() == 0


def test_bad_positions_and_slots_set_the_status_bit():
    g = R.geom("B", window=128, slot_ctx=512, n_slots=2)
    e = R.engine(g)
    kvk, kvv = e.alloc_kv_layer(False, fill=0)
    part = e.alloc_part(2, 100)
    for rows in (1, 8, 100):
        for p, s in ((-1, 0), (513 - rows, 0), (5, 2), (5, -1)):
            out = new_out(e, 1, rows, g.n_head, g.head_dim)
            q = torch.zeros(1, rows, g.n_head, g.head_dim, dtype=torch.float16, device=e.device)
            e.attn_sinks(out, q, kvk, kvv, e.sinks(4), R.ids([p], e), part, rows=rows, kslot=R.ids([s], e), is_swa=False)
            torch.cuda.synchronize()
            assert e.device_status() == 1 and torch.isnan(out).all(), (rows, p, s)


def test_an_unmapped_page_that_is_needed_sets_the_status_bit():
    """Pages between the sinks and the window may be missing, those the rows see may not (page 0 is read in their place)."""
    g = R.geom("B", window=128, slot_ctx=1024)
    e = R.engine(g)
    q, k, v = R.draw(g, 900, 100, 3)
    recs = [R.quantised(g, k, v)]
    for rows in (1, 8, 100):
        for page, status in ((3, 0), (0, 1), (6, 1)):
            pg = R.Paged(e, recs, 0, 128, 5, skip=lambda i, p: p == page)
            out = new_out(e, 1, rows, g.n_head, g.head_dim)
            e.attn_sinks_paged(out, dev_q(e, q[None, :rows]), pg.desc, e.sinks(4), R.ids([900 - rows], e), e.alloc_part(1, rows),
                               rows=rows)
            torch.cuda.synchronize()
            assert e.device_status() == status, (rows, page)


def test_positions_at_the_end_of_32_bits():
    """A ring's positions only grow: the last ones the call takes, and those it refuses."""
    g = R.geom("B", window=128, slot_ctx=512)
    e = R.engine(g)
    last = 2 ** 31 - 1025
    for rows in (1, 8, 100):
        q, k, v = R.draw(g, 256, rows, rows)
        kr, vr = R.quantised(g, k, v)
        # the ring's 256 slots, and sinks from another time; what the rows see is put in order for the plain form
        kvk, kvv = e.alloc_kv_layer(True, fill=0)
        sk, bk, bv = e.alloc_sinks(4)
        for buf, s, r in ((kvk, bk, kr), (kvv, bv, vr)):
            buf.view(g.n_kv, 256, g.rec).copy_(torch.from_numpy(r.copy()))
            s.view(g.n_kv, sk.cap, g.rec)[:, :4].copy_(torch.from_numpy(r[:, 100:104].copy()))
        out = new_out(e, 1, rows, g.n_head, g.head_dim)
        part = e.alloc_part(1, rows)
        e.attn_sinks(out, dev_q(e, q[None]), kvk, kvv, sk, R.ids([last], e), part, rows=rows)
        torch.cuda.synchronize()
        assert e.device_status() == 0
        seen = np.r_[100:104, (np.arange(last + 1 - 128, last + rows) % 256)]
        # 4 sinks, then 128 + rows - 1 keys of the ring: rows at positions 4 + 127 ... of that sequence, window 128
        want = R.attend64(g, q, kr[:, seen], vr[:, seen], 131, 4, 128)
        R.assert_attention(to_np(out)[0], want, g, vr, f"rows {rows}")
        out = new_out(e, 1, rows, g.n_head, g.head_dim)
        e.attn_sinks(out, dev_q(e, q[None]), kvk, kvv, sk, R.ids([last + 1], e), part, rows=rows)
        torch.cuda.synchronize()
        assert e.device_status() == 1 and torch.isnan(out).all()


def test_a_capacity_that_ends_inside_a_tile():
    """slot_ctx need only be even: the last tile of a partition is shorter, and what follows is another slot's."""
    g = R.geom("B", window=128, slot_ctx=634, n_slots=3)
    for name in ("B", "R"):
        g = R.geom(name, window=128, slot_ctx=634, n_slots=3)
        e = R.engine(g)
        for rows in (1, 8, 34):
            p = 634 - rows
            q, k, v = R.draw(g, 634, rows, rows)
            recs = R.quantised(g, k, v)
            kvk, kvv = e.alloc_kv_layer(False, fill=0x7F)
            for buf, t in ((kvk, 0), (kvv, 1)):
                R.put(e, buf, {1: recs}, False, t)
            qd, pos, slot = dev_q(e, q[None]), R.ids([p], e), R.ids([1], e)
            out, out2 = new_out(e, 1, rows, g.n_head, g.head_dim), new_out(e, 1, rows, g.n_head, g.head_dim)
            e.attn_sinks(out, qd, kvk, kvv, e.sinks(70), pos, e.alloc_part(1, rows), rows=rows, kslot=slot, is_swa=False)
            score = torch.full((3, g.n_kv, 634), 5.0, device=e.device)
            e.attn_track(out2, score, None, qd, kvk, kvv, pos, e.alloc_track_part(1, rows, 634), rows=rows, kslot=slot)
            torch.cuda.synchronize()
            assert e.device_status() == 0
            R.assert_attention(to_np(out)[0], R.attend64(g, q, *recs, p, 70, 128), g, recs[1], f"sinks {name} {rows}")
            R.assert_attention(to_np(out2)[0], R.attend64(g, q, *recs, p), g, recs[1], f"track {name} {rows}")
            sc = score.cpu().numpy()
            R.assert_scores(sc[1], R.score64(g, q, recs[0], p, None), g, q, recs[0], p, f"scores {name} {rows}")
            assert (sc[[0, 2]] == 5.0).all()


def test_refusals():
    from bruce_engine_b200 import capi
    g = R.geom("B", window=128, slot_ctx=512, n_slots=2)
    e = R.engine(g)
    ring, full = e.alloc_kv_layer(True, fill=0), e.alloc_kv_layer(False, fill=0)
    sk, bk, bv = e.alloc_sinks(4)
    part = e.alloc_part(2, 512)

    def call(rows=1, n=1, sinks=sk, cache=ring, is_swa=True, pos=None, q=None):
        q = torch.zeros(n, rows, g.n_head, g.head_dim, dtype=torch.float16, device=e.device) if q is None else q
        e.attn_sinks(torch.empty_like(q), q, *cache, sinks, R.ids([5] * n, e) if pos is None else pos, part, rows=rows,
                     kslot=R.ids(range(n), e), is_swa=is_swa)

    call()
    for code, kw in ((capi.ERR_ARG, dict(sinks=e.sinks(4))),                       # a ring needs the buffers
                     (capi.ERR_ARG, dict(cache=full, is_swa=False)),               # a full cache has none
                     (capi.ERR_ARG, dict(sinks=capi.CSinks(bk.data_ptr(), bv.data_ptr(), 129, 128))),
                     (capi.ERR_ARG, dict(sinks=capi.CSinks(bk.data_ptr(), bv.data_ptr(), -1, 128))),
                     (capi.ERR_ARG, dict(sinks=capi.CSinks(bk.data_ptr(), bv.data_ptr(), 4, 64))),
                     (capi.ERR_ARG, dict(sinks=capi.CSinks(bk.data_ptr() + 8, bv.data_ptr(), 4, 128))),
                     (capi.ERR_CAPACITY, dict(rows=40, n=2)),                      # a prompt chunk is one sequence
                     (capi.ERR_CAPACITY, dict(rows=129)),                          # ... of at most a window on a ring
                     (capi.ERR_CAPACITY, dict(rows=513, cache=full, sinks=e.sinks(4), is_swa=False))):
        with pytest.raises(capi.BattnError) as err:
            call(**kw)
        assert err.value.code == code, kw
    with pytest.raises(ValueError):
        call(q=torch.zeros(1, 1, g.n_head, g.head_dim, dtype=torch.float32, device=e.device))
    with pytest.raises(ValueError):
        call(q=torch.zeros(1, 1, g.head_dim, g.n_head, dtype=torch.float16, device=e.device).transpose(2, 3))
    with pytest.raises(ValueError):
        call(cache=(ring[0][:-1], ring[1]))
    with pytest.raises(ValueError):
        call(pos=torch.zeros(1, dtype=torch.int64, device=e.device))
    with pytest.raises(ValueError):
        e.sinks(4, bk)
    with pytest.raises(ValueError):
        e.sinks(4, bk, bv, cap=512)                                                # more than the buffers hold
    with pytest.raises(ValueError):                                                # a scratch buffer for a shorter call
        e.attn_sinks(torch.empty(1, 100, g.n_head, g.head_dim, dtype=torch.float16, device=e.device),
                     torch.zeros(1, 100, g.n_head, g.head_dim, dtype=torch.float16, device=e.device), *ring, sk, R.ids([5], e),
                     part[:4096], rows=100)
    n = __import__("ctypes").c_size_t()
    assert e.lib.battn_sinks_bytes(e.h, 100, n) == capi.ERR_ARG and e.lib.battn_sinks_bytes(e.h, 0, n) == capi.ERR_ARG
    torch.cuda.synchronize()
    assert e.device_status() == 0
