"""Early streaming (battn_set_early_kv_stream) of the calls with sinks and of the weight-accumulating ones, for active sequences:
behind the append of the same rows, and back to back on one scratch.  Every result is compared bit for bit with the option off,
and with 64 bits.  (battn_sinks_store is a launch that writes cache rows: a call behind it never streams early, so the ring
cases here are past their sink buffers and need no store.)"""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R
from tests.gpu_util import new_out, to_np

pytestmark = pytest.mark.gpu

STEPS = 4


class Stream:
    """n_seq sequences of `lens` cached positions and STEPS * rows rows to come, over one kind of cache."""

    def __init__(self, name, window, lens, rows, store, n_sink, seed):
        self.lens, self.rows, self.n_sink, self.window, self.store = lens, rows, n_sink, window, store
        n_seq, new = len(lens), STEPS * rows
        cap = max(lens) + new + 2
        cap += -cap % 128
        self.g = g = R.geom(name, window=window, slot_ctx=cap, n_slots=n_seq + 1)
        self.e = e = R.engine(g)
        self.order = np.random.default_rng(seed).permutation(n_seq + 1)[:n_seq]
        self.q, self.recs, ks, vs = [], [], [], []
        for i, p in enumerate(lens):
            q, k, v = R.draw(g, p + new, new, seed * 50 + i)
            self.q.append(q)
            self.recs.append(R.quantised(g, k, v))
            ks.append(k[p:])
            vs.append(v[p:])
        self.dq, self.dk, self.dv = (torch.from_numpy(np.stack(x)).to(e.device) for x in (self.q, ks, vs))
        self.dq = self.dq.to(e.q_torch)
        # per step its own tensors: nothing but the library's launches stands between the steps
        self.step = [[x[:, t * rows:(t + 1) * rows].contiguous() for x in (self.dq, self.dk, self.dv)] for t in range(STEPS)]
        self.pos = [R.ids([p + t * rows for p in lens], e) for t in range(STEPS)]
        self.ks = R.ids(self.order, e)
        self.reset()

    def reset(self):
        """The caches as they are before the first step."""
        g, e = self.g, self.e
        held = [[x[:, :p].copy() for x in r] for r, p in zip(self.recs, self.lens)]
        if self.store == "paged":
            self.pg = R.Paged(e, held, STEPS * self.rows, 128, 5)
            self.tab = torch.full((g.n_slots, self.pg.table.shape[1]), -1, dtype=torch.int32, device=e.device)
            self.tab[torch.from_numpy(self.order.copy()).long()] = self.pg.table
            self.pg.desc.table, self.pg.desc.n_tables = self.tab.data_ptr(), g.n_slots
            return
        ring = self.store == "ring"
        self.kv = e.alloc_kv_layer(ring, fill=0x7F)
        for t in range(2):
            R.put(e, self.kv[t], {int(s): held[i] for i, s in enumerate(self.order)}, ring, t)
        self.sk = e.sinks(self.n_sink)
        if ring:
            self.sk, *self.bufs = e.alloc_sinks(self.n_sink)
            assert min(self.lens) >= self.sk.cap
            for t in range(2):
                host = np.full((g.n_slots, g.n_kv, self.sk.cap, g.rec), 0x7F, dtype=np.uint8)
                for i, s in enumerate(self.order):
                    host[s] = held[i][t][:, :self.sk.cap]
                self.bufs[t].copy_(torch.from_numpy(host.reshape(-1)))

    def append(self, t):
        _, k, v = self.step[t]
        if self.store == "paged":
            self.e.kv_append_paged(self.pg.desc, k, v, self.pos[t], ktab=self.ks, rows=self.rows)
        else:
            self.e.qkv_prep_store(k, v, *self.kv, self.pos[t], kslot=self.ks, rows=self.rows, is_swa=self.store == "ring")

    def sinks(self, t, out, part):
        if self.store == "paged":
            self.e.attn_sinks_paged(out, self.step[t][0], self.pg.desc, self.e.sinks(self.n_sink), self.pos[t], part, rows=self.rows,
                                    ktab=self.ks)
        else:
            self.e.attn_sinks(out, self.step[t][0], *self.kv, self.sk, self.pos[t], part, rows=self.rows, kslot=self.ks,
                              is_swa=self.store == "ring")

    def track(self, t, out, score, part, fresh=False):
        given = None if fresh else score
        if self.store == "paged":
            self.e.attn_track_paged(out, score, given, self.step[t][0], self.pg.desc, self.pos[t], part, rows=self.rows, ktab=self.ks)
        else:
            self.e.attn_track(out, score, given, self.step[t][0], *self.kv, self.pos[t], part, rows=self.rows, kslot=self.ks)

    def new(self):
        return new_out(self.e, len(self.lens), self.rows, self.g.n_head, self.g.head_dim)

    def scores(self):
        cap = self.pg.desc.max_pages * 128 if self.store == "paged" else self.g.slot_ctx
        return torch.full((self.g.n_slots, self.g.n_kv, cap), float("nan"), device=self.e.device)


def _same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=77.0), torch.nan_to_num(b, nan=77.0))


ROWS = {"decode": ([1000, 517, 3001], 1), "one": ([3001], 1), "verify": ([1000, 517, 3001], 3), "chunk": ([2001], 100),
        "long chunk": ([1500], 256)}


@pytest.mark.parametrize("store", ["ring", "slots", "paged"])
@pytest.mark.parametrize("kind", list(ROWS))
@pytest.mark.parametrize("name", ["B", "R"])
def test_sinks_behind_the_append(name, kind, store):
    lens, rows = ROWS[kind]
    s = Stream(name, 256, lens, rows, store, 5, 3)
    got = []
    for early in (False, True):
        s.reset()
        s.e.set_early_kv_stream(early)
        part, outs = s.e.alloc_part(len(lens), rows), [s.new() for _ in range(STEPS)]
        torch.cuda.synchronize()
        for t in range(STEPS):
            s.append(t)
            s.sinks(t, outs[t], part)
        torch.cuda.synchronize()
        assert s.e.device_status() == 0
        got.append(outs)
    for t in range(STEPS):
        assert torch.equal(got[0][t], got[1][t]), t
        for i, p in enumerate(lens):
            at = p + t * rows
            seen = [x[:, :at + rows] for x in s.recs[i]]
            want = R.attend64(s.g, s.q[i][t * rows:(t + 1) * rows], *seen, at, 5, 256)
            R.assert_attention(to_np(got[1][t])[i], want, s.g, seen[1], f"{kind} {store} step {t} of {i}")


@pytest.mark.parametrize("store", ["slots", "paged"])
@pytest.mark.parametrize("kind", ["decode", "one", "chunk", "long chunk"])
@pytest.mark.parametrize("name", ["B", "R"])
def test_weights_behind_the_append_and_back_to_back(name, kind, store):
    """Per step: append, accumulate, then two more calls on the same scratch with nothing between them (the previous call's merge
    may still read its records and scores when the next one starts to stream)."""
    lens, rows = ROWS[kind]
    s = Stream(name, 256, lens, rows, store, 5, 4)
    got = []
    for early in (False, True):
        s.reset()
        s.e.set_early_kv_stream(early)
        part = s.e.alloc_track_part(len(lens), rows, sum(lens) + len(lens) * STEPS * rows)
        score, other = s.scores(), s.scores()
        for i, p in enumerate(lens):
            score[int(s.order[i]), :, :p] = 0.0
        outs, scs = [s.new() for _ in range(2 * STEPS)], []
        torch.cuda.synchronize()
        for t in range(STEPS):
            s.append(t)
            s.track(t, outs[2 * t], score, part)
            s.track(t, outs[2 * t + 1], other, part, fresh=True)
            s.track(t, outs[2 * t], score, part)                     # the rows count twice
        torch.cuda.synchronize()
        assert s.e.device_status() == 0
        got.append(outs + [score.clone(), other.clone()])
    for a, b in zip(*got):
        assert _same(a, b)
    last = STEPS - 1
    for i, p in enumerate(lens):
        at = p + last * rows
        q = s.q[i][last * rows:]
        R.assert_attention(to_np(got[1][2 * last])[i], R.attend64(s.g, q, *s.recs[i], at), s.g, s.recs[i][1], f"{kind} {store} of {i}")
        R.assert_scores(got[1][-1].cpu().numpy()[s.order[i], :, :at + rows], R.score64(s.g, q, s.recs[i][0], at, None), s.g, q,
                        s.recs[i][0], at, f"{kind} {store} weights of {i}")
        assert torch.equal(got[1][2 * last][i], got[1][2 * last + 1][i])
        # every step's own positions start from nothing in both of its calls; the earlier ones were given both calls' weights
        sc = got[1][-2].cpu().numpy()[s.order[i], :, :at + rows].astype(np.float64)
        want = np.zeros_like(sc)
        for t in range(STEPS):
            a = p + t * rows
            w = R.score64(s.g, s.q[i][t * rows:(t + 1) * rows], s.recs[i][0][:, :a + rows], a, None)
            want[:, :a] += 2 * w[:, :a]
            want[:, a:a + rows] = w[:, a:]
        # sums of positive terms, each within the relative bound of R.assert_scores: with sum |q k| below 60 and at most 3100
        # positions, 2 * 0.6932 * 16 * 2^-23 * 60 + 8 * 2^-22 + (1550 + 1024) * 2^-24 = 3.2e-4, and 8 additions at 2^-24
        assert np.isfinite(sc).all() and (np.abs(sc - want) <= 3.3e-4 * want + 1e-30).all()


def test_a_trim_between_early_steps():
    """accumulate -> trim -> append -> accumulate with early streaming: the call behind the append reads what the trim moved."""
    s = Stream("B", 256, [1000, 517, 3001], 1, "slots", 5, 6)
    got = []
    for early in (False, True):
        s.reset()
        s.e.set_early_kv_stream(early)
        part, ep = s.e.alloc_track_part(3, 1, 6000), s.e.alloc_evict_part(3)
        score = s.scores()
        kept = torch.zeros(3, s.g.n_kv, 300, dtype=torch.int32, device=s.e.device)
        outs, pos = [s.new() for _ in range(3)], s.pos[0].clone()
        torch.cuda.synchronize()
        s.append(0)
        s.track(0, outs[0], score, part, fresh=True)
        for t in range(2):
            s.e.evict(*s.kv, score, kept, pos, pos, ep, 300 - 50 * t, n_sink=4, n_recent=20, kslot=s.ks)
            q, k, v = s.step[t + 1]
            s.e.qkv_prep_store(k, v, *s.kv, pos, kslot=s.ks)
            s.e.attn_track(outs[t + 1], score, score, q, *s.kv, pos, part, kslot=s.ks)
        torch.cuda.synchronize()
        assert s.e.device_status() == 0 and pos.tolist() == [250] * 3
        got.append(outs + [score, kept.clone()] + [x.clone() for x in s.kv])
    for a, b in zip(*got):
        assert _same(a, b) if a.is_floating_point() else torch.equal(a, b)
