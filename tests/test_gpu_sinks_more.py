"""Sink buffers at their limits, groups of every size, early streaming and unrounded queries of the calls with sinks."""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R
from tests.gpu_util import dev_q, new_out, to_np

pytestmark = pytest.mark.gpu


def test_sink_buffers_whose_words_pass_32_bits():
    """cap is any multiple of 128: positions whose 8-byte words, counted from their head's start, pass 2 ** 31."""
    cap = 1 << 26                                                    # 34 words a record: 2 ** 31 words are 63.2 million
    g = R.geom("R", window=128, slot_ctx=512, n_head=4, n_kv=1)
    assert (cap - 1) * (g.rec // 8) > 2 ** 31
    e = R.engine(g)
    ring = [torch.randint(0, 60, (e.kv_layer_bytes(True),), dtype=torch.uint8, device=e.device) for _ in range(2)]
    bufs = [torch.empty(cap * g.rec, dtype=torch.uint8, device=e.device) for _ in range(2)]
    sk = e.sinks(4, *bufs)
    assert sk.cap == cap
    for rows, p in ((1, cap - 1), (1, 2 ** 31 // 34 + 1), (40, cap - 40), (40, cap - 7), (1, cap), (3, 0)):
        held = min(rows, cap - p)
        for b in bufs:
            b.view(cap, g.rec)[max(0, p - 2):p + rows].fill_(0x7F)
        e.sinks_store(*ring, sk, R.ids([p], e), rows=rows)
        torch.cuda.synchronize()
        assert e.device_status() == 0
        for b, r in zip(bufs, ring):
            at = torch.arange(p, p + max(held, 0), device=e.device)
            assert torch.equal(b.view(cap, g.rec)[p:p + max(held, 0)], r.view(2 * g.window, g.rec)[at % (2 * g.window)])
            assert (b.view(cap, g.rec)[max(0, p - 2):p] == 0x7F).all()


# ---- groups of every size -------------------------------------------------------------------------------------------------
def _group(monkeypatch, group):
    """The geometries of the other tests with `group` query heads per kv head."""
    plain = R.geom
    monkeypatch.setattr(R, "geom", lambda name, **kw: plain(name, n_head=2 * group, n_kv=2, **kw))


@pytest.mark.parametrize("group", [2, 3, 5, 6, 7])
@pytest.mark.parametrize("name", ["B", "R"])
def test_groups_of_every_size(monkeypatch, name, group):
    from tests.test_gpu_sinks import _case as sinks
    from tests.test_gpu_track import _case as track
    _group(monkeypatch, group)
    for store in ("ring", "slots", "paged"):
        sinks(name, 128, [0, 3, 127, 128, 191, 300, 1001], 1, 5, store, 7)
        for rows in (2, 3, 4, 5, 8):
            if rows * group <= 32:
                sinks(name, 256, [0, 2, 252, 256, 700], rows, 5, store, 8 + rows)
    for store in ("slots", "paged"):
        for how in ("add", "same", "none"):
            track(name, [0, 1, 63, 64, 500, 2047, 3001], 1, store, 3, how)
        track(name, [9000], 1, store, 4, "same")
        if 128 % group == 0:
            sinks(name, 256, [900], 90, 64, store, 5)
            track(name, [900], 90, store, 5, "same")


@pytest.mark.parametrize("group", [3, 5, 6, 7])
def test_prompt_chunks_refuse_groups_that_do_not_divide_a_tile(monkeypatch, group):
    from bruce_engine_b200 import capi
    _group(monkeypatch, group)
    g = R.geom("B", window=128, slot_ctx=512)
    e = R.engine(g)
    cache, score = e.alloc_kv_layer(False, fill=0), torch.full((1, g.n_kv, 512), 5.0, device=e.device)
    q = torch.zeros(1, 64, g.n_head, g.head_dim, dtype=torch.float16, device=e.device)
    out, pos = new_out(e, 1, 64, g.n_head, g.head_dim), R.ids([100], e)
    for call in (lambda: e.attn_sinks(out, q, *cache, e.sinks(4), pos, e.alloc_part(1, 64), rows=64, is_swa=False),
                 lambda: e.attn_track(out, score, score, q, *cache, pos, e.alloc_track_part(1, 64, 512), rows=64)):
        with pytest.raises(capi.BattnError) as err:
            call()
        assert err.value.code == capi.ERR_ARG
    torch.cuda.synchronize()
    assert e.device_status() == 0 and torch.isnan(out).all() and (score == 5.0).all()


# ---- fp32 queries ---------------------------------------------------------------------------------------------------------
def _attend_and_slack(g, q, krec, vrec, p0, window, n_sink):
    """Attention in 64 bits on the queries as given, the weights, and what rounding the queries to fp16 may move the output.

    A query component moves by at most U of itself, so the score of key k by at most e_k = U sum_d |q_d k_d| * scale, and the
    output, sum w e^x v / sum w e^x with |x_k| <= e_k <= E, by at most (sum_k w_k (e_k + E^2) |v_k - out|) / (1 - E)
    (|e^x - 1| <= |x| + x^2 for |x| < 1, and the denominator is at least e^-E >= 1 - E)."""
    rows, n = q.shape[0], p0 + q.shape[0]
    w = R.weights64(g, q, krec, p0, n_sink, window)
    kd, vd = (torch.from_numpy(R.values(x[:, :n], g.head_dim)).cuda() for x in (krec, vrec))
    qd = torch.from_numpy(q.astype(np.float64)).cuda()
    scale = g.head_dim ** -0.5
    out, slack, big = np.zeros((2, rows, g.n_head, g.head_dim)), 0.0, 0.0
    for h in range(g.n_head):
        k, v = kd[h // g.group], vd[h // g.group]
        e = R.U * scale * (qd[:, h].abs() @ k.abs().T)
        top = float(torch.where(w[h] > 0, e, 0.0).max())
        big = max(big, top)
        for r in range(rows):
            o = w[h, r] @ v
            out[0, r, h] = o.cpu().numpy()
            out[1, r, h] = ((w[h, r] * (e[r] + top * top)) @ (v - o).abs() / (1 - top)).cpu().numpy()
    return out[0], out[1], w, big


@pytest.mark.parametrize("name", ["B32", "R"])
@pytest.mark.parametrize("rows", [1, 7, 40])
def test_what_rounding_fp32_queries_costs(name, rows):
    """Queries that fp16 does not hold: outputs and weights against 64 bits on the queries as given."""
    from bruce_engine_b200.layout import F32
    g = R.geom(name, window=512, slot_ctx=2048, q_dtype=F32)
    e = R.engine(g)
    p = 1500
    _, k, v = R.draw(g, p + rows, rows, rows)
    q = (1.5 * np.random.default_rng(rows).standard_normal((rows, g.n_head, g.head_dim))).astype(np.float32)
    assert (q != q.astype(np.float16)).mean() > 0.9
    recs = R.quantised(g, k, v)
    kvk, kvv = e.alloc_kv_layer(False, fill=0x7F)
    for t, buf in enumerate((kvk, kvv)):
        R.put(e, buf, {0: recs}, False, t)
    qd, pos = torch.from_numpy(q[None]).to(e.device), R.ids([p], e)
    score = torch.full((1, g.n_kv, 2048), float("nan"), device=e.device)
    outs = [new_out(e, 1, rows, g.n_head, g.head_dim) for _ in range(2)]
    e.attn_sinks(outs[0], qd, kvk, kvv, e.sinks(4), pos, e.alloc_part(1, rows), rows=rows, is_swa=False)
    e.attn_track(outs[1], score, None, qd, kvk, kvv, pos, e.alloc_track_part(1, rows, p + rows), rows=rows)
    torch.cuda.synchronize()
    assert e.device_status() == 0
    vmax = np.repeat(np.abs(R.values(recs[1], g.head_dim)).max(1), g.group, axis=0)[None]
    for out, window, n_sink in ((outs[0], 512, 4), (outs[1], None, None)):
        want, slack, w, big = _attend_and_slack(g, q, *recs, p, window, n_sink)
        # R.assert_attention's bound for queries that fp16 holds, plus the rounding of these
        assert (np.abs(to_np(out)[0].astype(np.float64) - want) <= 3.5 * R.U * vmax + R.U * np.abs(want) + slack).all()
    # a weight moves by a factor between e^(-2 E) and e^(2 E); beside it R.assert_scores' bound, below 1e-3 for these sizes
    sc = w.sum(1).reshape(g.n_kv, g.group, -1).sum(1).cpu().numpy()
    assert (np.abs(score[0, :, :p + rows].cpu().numpy() - sc) <= (np.exp(2 * big) - 1 + 1e-3) * sc + 1e-30).all()
