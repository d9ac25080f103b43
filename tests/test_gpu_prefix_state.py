"""A conversation that starts behind another one's cached prefix: what is copied beside the records -- sink buffers of a window
layer, accumulated scores -- by the engine's prefix copy or by the host as battn.h says, over what the slot's (or table row's)
previous conversation left there."""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R
from tests.gpu_util import dev_q, new_out, to_np

pytestmark = pytest.mark.gpu


def _fill(buf, layout, slot, rec):
    """Records [n_kv][n][record] at the front of a slot of a buffer laid out [slot][n_kv][positions][record]."""
    buf.view(*layout)[slot, :, :rec.shape[1]].copy_(torch.from_numpy(rec.copy()))


@pytest.mark.parametrize("by", ["engine", "host"])
@pytest.mark.parametrize("name", ["B", "R"])
@pytest.mark.parametrize("shared", [30, 128, 200, 700])
def test_sinks_of_a_copied_prefix(name, shared, by):
    """Slot 1 held another conversation; a prefix of slot 0's is copied into it, then rows are appended and attended."""
    window, n_sink, new = 128, 5, 40
    g = R.geom(name, window=window, slot_ctx=1024, n_slots=2)
    e = R.engine(g)
    q, k, v = R.draw(g, shared + new, new, shared)
    recs = R.quantised(g, k, v)
    _, k2, v2 = R.draw(g, 300, 1, shared + 1)
    old = R.quantised(g, k2, v2)
    ring = e.alloc_kv_layer(True, fill=0x7F)
    sk, *bufs = e.alloc_sinks(n_sink)
    layout = (2, g.n_kv, sk.cap, g.rec)
    for t in range(2):
        R.put(e, ring[t], {0: [x[:, :shared] for x in recs], 1: old}, True, t)
        _fill(bufs[t], layout, 0, recs[t][:, :min(shared, sk.cap)])
        _fill(bufs[t], layout, 1, old[t][:, :sk.cap])
    e.kv_copy_prefix(*ring, 0, 1, shared, is_swa=True, sinks=sk if by == "engine" else None)
    n = min(shared, sk.cap)
    for t, b in enumerate(bufs):
        x = b.view(*layout)
        if by == "host":
            x[1, :, :n].copy_(x[0, :, :n])
        assert torch.equal(x[1, :, :n], x[0, :, :n]) and (x[1, :, n:].cpu().numpy() == old[t][:, n:sk.cap]).all()
    slot, part = R.ids([1], e), e.alloc_part(1, new)
    at = shared
    for rows in (new - 1, 1):                                        # a chunk, then a token
        i = slice(at - shared, at - shared + rows)
        kd, vd = (torch.from_numpy(x[at:at + rows]).to(e.device) for x in (k, v))
        pos, out = R.ids([at], e), new_out(e, 1, rows, g.n_head, g.head_dim)
        e.qkv_prep_store(kd, vd, *ring, pos, kslot=slot, rows=rows, is_swa=True)
        e.sinks_store(*ring, sk, pos, kslot=slot, rows=rows)
        e.attn_sinks(out, dev_q(e, q[None, i]), *ring, sk, pos, part, rows=rows, kslot=slot)
        torch.cuda.synchronize()
        assert e.device_status() == 0
        seen = [x[:, :at + rows] for x in recs]
        R.assert_attention(to_np(out)[0], R.attend64(g, q[i], *seen, at, n_sink, window), g, seen[1], f"{rows} rows behind {shared}")
        at += rows


@pytest.mark.parametrize("store", ["slots", "paged"])
@pytest.mark.parametrize("counted", [True, False])
def test_scores_of_a_copied_or_shared_prefix(store, counted):
    """The prefix's accumulated weights go with it (or, where the new conversation is to count for itself, are set to nothing);
    partition 1's own were another conversation's."""
    shared, rows = 384, 20
    g = R.geom("B", slot_ctx=512, n_slots=2)
    e = R.engine(g)
    q, k, v = R.draw(g, shared + rows, rows, 3)
    recs = R.quantised(g, k, v)
    held = [x[:, :shared] for x in recs]
    rng = np.random.default_rng(4)
    score = torch.from_numpy(rng.random((2, g.n_kv, 512), dtype=np.float32)).to(e.device)
    first = score[0].cpu().numpy().copy()
    kd, vd = (torch.from_numpy(x[shared:]).to(e.device) for x in (k, v))
    sel, pos = R.ids([1], e), R.ids([shared], e)
    if store == "slots":
        kv = e.alloc_kv_layer(False, fill=0x7F)
        for t in range(2):
            R.put(e, kv[t], {0: held}, False, t)
        e.kv_copy_prefix(*kv, 0, 1, shared, score=score if counted else None)
    else:
        # three pages of row 0, shared by row 1, which appends into a page of its own
        tab = torch.tensor([[4, 0, 2, -1], [4, 0, 2, 1]], dtype=torch.int32, device=e.device)
        desc, *pools = e.alloc_pages(5, 128, tab, fill=0x7F)
        for t in range(2):
            for p, page in enumerate((4, 0, 2)):
                pools[t].view(5, g.n_kv, 128, g.rec)[page].copy_(torch.from_numpy(held[t][:, 128 * p:128 * (p + 1)].copy()))
    if store == "paged" or not counted:
        score[1, :, :shared] = score[0, :, :shared] if counted else 0.0
    for n in (rows - 1, 1):
        i = slice(int(pos[0]) - shared, int(pos[0]) - shared + n)
        out, part = new_out(e, 1, n, g.n_head, g.head_dim), e.alloc_track_part(1, n, 512)
        qd = dev_q(e, q[None, i])
        if store == "slots":
            e.qkv_prep_store(kd[i].contiguous(), vd[i].contiguous(), *kv, pos, kslot=sel, rows=n)
            e.attn_track(out, score, score, qd, *kv, pos, part, rows=n, kslot=sel)
        else:
            e.kv_append_paged(desc, kd[i].contiguous(), vd[i].contiguous(), pos, ktab=sel, rows=n)
            e.attn_track_paged(out, score, score, qd, desc, pos, part, rows=n, ktab=sel)
        pos += n
    torch.cuda.synchronize()
    assert e.device_status() == 0
    before = first.astype(np.float64) if counted else np.zeros((g.n_kv, 512))
    mid = R.score64(g, q[:rows - 1], recs[0][:, :-1], shared, before)
    want = R.score64(g, q[rows - 1:], recs[0], shared + rows - 1, mid)
    got = score.cpu().numpy()
    # (two accumulations: twice the bound of one)
    R.assert_scores(want + (got[1, :, :shared + rows] - want) / 2, want, g, q, recs[0], shared, "scores behind a prefix")
    assert (got[0] == first).all()


def test_refusals():
    g = R.geom("B", window=128, slot_ctx=512, n_slots=2)
    e = R.engine(g)
    ring, full = e.alloc_kv_layer(True, fill=0), e.alloc_kv_layer(False, fill=0)
    sk, bk, bv = e.alloc_sinks(4)
    score = torch.zeros(2, g.n_kv, 512, device=e.device)
    one = e.sinks(4, bk.view(2, -1)[0], bv.view(2, -1)[0], cap=sk.cap)
    for cache, kw in ((ring, dict(is_swa=True, sinks=one)), (ring, dict(is_swa=True, sinks=e.sinks(4))), (full, dict(sinks=sk)),
                      (ring, dict(is_swa=True, score=score)), (full, dict(score=score[:1])), (full, dict(score=score.double()))):
        with pytest.raises(ValueError):
            e.kv_copy_prefix(*cache, 0, 1, 100, **kw)
    torch.cuda.synchronize()
    assert e.device_status() == 0
