"""Positions that no cache holds, up to the last 32-bit one: the attention calls set BATTN_DEV_BAD_POSITION, write nothing for
that sequence, and give the other sequences of the call what they get beside an idle one."""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R
from tests.gpu_util import dev_q, new_out

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1
BAD = 1


def _far(rows, ring):
    """The ends of 32 bits, with and without the rows; a ring takes rows that end at 2 ** 31 - 257."""
    p = {TOP, TOP - 1, TOP - rows, TOP - rows + 1, TOP - rows - 127, TOP - rows - 255}
    return sorted(p) if ring else sorted(p | {TOP - rows - 256, 513 - rows})


def _calls(e, rows, store):
    """(name, fn(out, q, pos, kslot)) of every attention call that takes `rows` rows of one sequence over that cache."""
    g = e.geom
    sc = torch.full((2, g.n_kv, 512), 5.0, device=e.device)
    if store == "paged":
        tab = torch.arange(8, dtype=torch.int32, device=e.device).reshape(2, 4)
        desc, pk, pv = e.alloc_pages(8, 128, tab, fill=1)
        part, tp = e.alloc_part(1, rows), e.alloc_track_part(1, rows, 600)
        keep = (tab, pk, pv)
        yield "plain", lambda o, q, p, s: e.attn_paged(o, q, desc, p, part, rows=rows, ktab=s), None, keep
        yield "sinks", lambda o, q, p, s: e.attn_sinks_paged(o, q, desc, e.sinks(4), p, part, rows=rows, ktab=s), None, keep
        yield "track", lambda o, q, p, s: e.attn_track_paged(o, sc, sc, q, desc, p, tp, rows=rows, ktab=s), sc, keep
        return
    ring = store == "ring"
    kvk, kvv = e.alloc_kv_layer(ring, fill=1)
    part = e.alloc_part(1, rows)
    ns = 2 if rows > 8 else 4
    xp = torch.empty(e.exact_workspace_bytes(1, rows, ns), dtype=torch.uint8, device=e.device)
    yield "plain", lambda o, q, p, s: e.launch_attn_m(o, q, kvk, kvv, p, part, rows, is_swa=ring), None, None
    yield "exact", lambda o, q, p, s: e.attn_exact(o, q, kvk, kvv, p, xp, 1, rows, ns, is_swa=ring, kslot=s), None, None
    if rows == 1:
        kv = torch.zeros(1, 1, g.n_kv, g.head_dim, device=e.device)
        yield "append", lambda o, q, p, s: e.decode_append(o, q, kv, kv, kvk, kvv, p, part, kslot=s, is_swa=ring), None, None
    sk, bk, bv = e.alloc_sinks(4) if ring else (e.sinks(4), None, None)
    yield "sinks", lambda o, q, p, s: e.attn_sinks(o, q, kvk, kvv, sk, p, part, rows=rows, kslot=s, is_swa=ring), None, (bk, bv)
    if not ring:
        tp = e.alloc_track_part(1, rows, 600)
        yield "track", lambda o, q, p, s: e.attn_track(o, sc, sc, q, kvk, kvv, p, tp, rows=rows, kslot=s), sc, None


@pytest.mark.parametrize("store", ["slots", "ring", "paged"])
@pytest.mark.parametrize("name", ["B", "R"])
def test_positions_whose_rows_pass_32_bits(name, store):
    g = R.geom(name, window=128, slot_ctx=512, n_slots=2)
    e = R.engine(g)
    slot = R.ids([1], e)
    for rows in (1, 2, 8, 40, 128):
        q = torch.zeros(1, rows, g.n_head, g.head_dim, dtype=e.q_torch, device=e.device)
        for what, call, score, _ in _calls(e, rows, store):
            for p in _far(rows, store == "ring"):
                out = new_out(e, 1, rows, g.n_head, g.head_dim)
                call(out, q, R.ids([p], e), slot)
                torch.cuda.synchronize()
                assert e.device_status() == BAD, (what, rows, p)
                # (a plain prompt chunk is always active: what its merge makes of absent records is not defined)
                if what != "plain" or rows <= 8:
                    assert torch.isnan(out).all(), (what, rows, p)
                assert score is None or (score == 5.0).all(), (what, rows, p)


def test_one_split_of_a_prompt_chunk_has_no_records_to_write():
    """512 rows of 32 / 8 heads: a CTA per (M tile, kv head), no split records."""
    g = R.geom("B", slot_ctx=1024, n_slots=2)
    e = R.engine(g)
    kvk, kvv = e.alloc_kv_layer(False, fill=1)
    q = torch.zeros(1, 512, g.n_head, g.head_dim, dtype=torch.float16, device=e.device)
    score, part, tp = torch.full((2, g.n_kv, 1024), 5.0, device=e.device), e.alloc_part(1, 512), e.alloc_track_part(1, 512, 1024)
    slot = R.ids([1], e)
    for p in (TOP, TOP - 511, TOP - 512, 513):
        for call in (lambda o: e.attn_track(o, score, score, q, kvk, kvv, R.ids([p], e), tp, rows=512, kslot=slot),
                     lambda o: e.attn_sinks(o, q, kvk, kvv, e.sinks(4), R.ids([p], e), part, rows=512, kslot=slot, is_swa=False),
                     lambda o: e.launch_attn_m(o, q, kvk, kvv, R.ids([p], e), part, 512)):
            out = new_out(e, 1, 512, g.n_head, g.head_dim)
            call(out)
            torch.cuda.synchronize()
            assert e.device_status() == BAD and torch.isnan(out).all() and (score == 5.0).all(), p


@pytest.mark.parametrize("rows", [1, 3, 8])
def test_the_other_sequences_of_a_batch(rows):
    """Good sequences before, between and behind bad ones: bit for bit what they give when the bad ones are idle."""
    g = R.geom("B", window=128, slot_ctx=2048, n_slots=6)
    e = R.engine(g)
    kvk, kvv = (torch.randint(0, 60, (e.kv_layer_bytes(False),), dtype=torch.uint8, device=e.device) for _ in range(2))
    rng = np.random.default_rng(rows)
    q = dev_q(e, rng.standard_normal((6, rows, g.n_head, g.head_dim)).astype(np.float32))
    ks, part = R.ids([3, 0, 5, 1, 4, 2], e), e.alloc_part(6, rows)
    good = [1500, 700, 1900, 64]
    for far in (TOP, TOP - rows + 1, TOP - rows, TOP - rows - 127):
        pos = R.ids([good[0], far, good[1], good[2], far, good[3]], e)
        act = R.ids([1, 0, 1, 1, 0, 1], e)
        calls = [lambda o, a: e.launch_attn_ms(o, q, kvk, kvv, pos, ks, a, part, 6, rows_per_seq=rows),
                 lambda o, a: e.attn_sinks(o, q, kvk, kvv, e.sinks(4), pos, part, rows=rows, kslot=ks, act=a, is_swa=False)]
        if rows == 1:
            tp = e.alloc_track_part(6, 1, sum(good) + 6)
            sc = torch.full((6, g.n_kv, 2048), 5.0, device=e.device)
            calls.append(lambda o, a: e.attn_track(o, sc, None, q, kvk, kvv, pos, tp, kslot=ks, act=a))
        for i, call in enumerate(calls):
            got = []
            for a in (act, None):
                out = new_out(e, 6, rows, g.n_head, g.head_dim)
                if i == 2:
                    sc.fill_(5.0)
                call(out, a)
                torch.cuda.synchronize()
                assert e.device_status() == (BAD if a is None else 0)
                got.append([out.clone()] + ([sc.clone()] if i == 2 else []))
            assert torch.isnan(got[0][0][[1, 4]]).all() and torch.isfinite(got[0][0][[0, 2, 3, 5]]).all()
            for x, y in zip(*got):
                assert torch.equal(torch.nan_to_num(x, nan=7.0), torch.nan_to_num(y, nan=7.0)), (i, far)


@pytest.mark.parametrize("name", ["B", "R"])
def test_a_refused_prompt_chunk_keeps_the_order_of_the_stream(name):
    """With early streaming, append -> chunk that ends past the cache -> decode over the rows that were appended: the refused
    chunk's launches still stand behind the append, so the decode reads its rows, as without early streaming."""
    cap, rows = 4096, 512
    g = R.geom(name, window=1024, slot_ctx=cap)
    e = R.engine(g)
    rng = np.random.default_rng(3)
    q1, qc = (dev_q(e, rng.standard_normal((1, r, g.n_head, g.head_dim)).astype(np.float32)) for r in (1, rows))
    kvk, kvv = e.alloc_kv_layer(False, fill=1)
    part, first, last = e.alloc_part(1, rows), R.ids([cap - 400], e), R.ids([cap - 1], e)
    junk = new_out(e, 1, rows, g.n_head, g.head_dim)
    for t in range(20):
        kv = torch.randn(2, rows, g.n_kv, g.head_dim, device=e.device)
        got = []
        for early in (True, False):
            kvk.fill_(1)
            kvv.fill_(1)
            torch.cuda.synchronize()
            out = new_out(e, 1, 1, g.n_head, g.head_dim)
            e.set_early_kv_stream(early)
            e.qkv_prep_store(kv[0], kv[1], kvk, kvv, first, rows=rows)
            e.launch_attn_m(junk, qc, kvk, kvv, first, part, rows)
            e.launch_attn_m(out, q1, kvk, kvv, last, part, 1)
            torch.cuda.synchronize()
            assert e.device_status() == BAD
            got.append(out)
        assert torch.isfinite(got[0]).all() and torch.equal(*got), t
