"""Accumulated weights at long contexts, held to their 2-norm distance from 64 bits beside the bound per element, whose
summation term alone passes 1e-3 at 40000 positions (bounded_ref.assert_scores).

One row: an exponent of up to 2^4 in log2 units carries a few independent roundings of 2^-24 of itself (fp32 sums of four or eight
scaled blocks), the denominator's sum about sqrt(n / 3) of them: well below ONE_ROW.

A chunk: the scores are formed on the tensor core in N = 2 * head_dim / 16 accumulation steps (K has two parts), each of which
drops what lies below the last of 24 bits of a running sum of up to X, the largest score that carries weight: an error between 0
and N 2^-23 X, always towards zero, in the exponent and, averaged over the keys, in the normaliser.  Their difference is at most
the same, and a weight moves by it times ln 2: 2.1e-5 at head_dim 128 and X = 2^4, twice that at 256.  It is not averaged away by more
rows, as the large scores all lose."""
import numpy as np
import pytest
import torch

from tests import bounded_ref as R
from tests.gpu_util import dev_q, new_out

pytestmark = pytest.mark.gpu

ONE_ROW = 1e-6


def _weights(name, lens, rows, seed):
    """Accumulated weights of rows behind `lens` positions, and their value in 64 bits: [n_kv][positions] per sequence."""
    g = R.geom(name, slot_ctx=max(lens) + rows + (rows & 1) + (max(lens) & 1), n_slots=len(lens))
    e = R.engine(g)
    q, recs = [], []
    for i, p in enumerate(lens):
        qq, k, v = R.draw(g, p + rows, rows, seed + i)
        q.append(qq)
        recs.append(R.quantised(g, k, v))
    kvk, kvv = e.alloc_kv_layer(False, fill=0x7F)
    for t, buf in enumerate((kvk, kvv)):
        R.put(e, buf, dict(enumerate(recs)), False, t)
    score = torch.full((len(lens), g.n_kv, g.slot_ctx), float("nan"), device=e.device)
    n = sum(lens) + len(lens) * rows
    e.attn_track(new_out(e, len(lens), rows, g.n_head, g.head_dim), score, None, dev_q(e, np.stack(q)), kvk, kvv, R.ids(lens, e),
                 e.alloc_track_part(len(lens), rows, n), rows=rows, kslot=R.ids(range(len(lens)), e))
    torch.cuda.synchronize()
    assert e.device_status() == 0
    got = score.cpu().numpy().astype(np.float64)
    for i, p in enumerate(lens):
        yield g, got[i, :, :p + rows], R.score64(g, q[i], recs[i][0], p, None), (q[i], recs[i][0], p)


def _ratio(got, want):
    return np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)


def _limit(g, q, krec, p):
    if len(q) == 1:
        return ONE_ROW
    w = R.weights64(g, q, krec, p)                               # scores that carry weight: within a factor 100 of the largest
    x = 0.0
    for h in range(g.n_head):
        k = torch.from_numpy(R.values(krec[h // g.group], g.head_dim)).cuda()
        s = torch.from_numpy(q[:, h].astype(np.float64)).cuda() @ k.T * (g.head_dim ** -0.5 * np.log2(np.e))
        x = max(x, float(torch.where(w[h] >= 0.01 * w[h].amax(-1, keepdim=True), s.abs(), 0.0).max()))
    return 2 * g.head_dim / 16 * 2.0 ** -23 * x * np.log(2.0) + ONE_ROW


@pytest.mark.parametrize("name,lens,rows", [("B", [16000], 1), ("B", [40001], 1), ("B", [3001, 30000, 9000], 1), ("B8", [20000], 1),
                                            ("R", [40001], 1), ("R", [3001, 16000], 1), ("B", [16000], 8), ("B", [16000], 384),
                                            ("R", [16000], 40), ("R16", [9000], 200)])
def test_weights_in_the_2_norm(name, lens, rows):
    for g, got, want, given in _weights(name, lens, rows, 5):
        r, limit = _ratio(got, want), _limit(g, *given)
        assert limit < 6e-5 and (r <= limit).all(), (name, lens, rows, r.max(), limit)


def test_the_limit_tells_a_denominator_of_rounded_weights():
    """The planted mistake, in the 64-bit form: dividing by the sum of fp16-rounded weights is outside the limit of one row."""
    for g, got, want, (q, krec, p) in _weights("B", [16000], 1, 5):
        w = R.weights64(g, q, krec, p)[:, 0].cpu().numpy()
        w /= w.max(1, keepdims=True)
        bad = (w / w.astype(np.float16).astype(np.float64).sum(1, keepdims=True)).reshape(g.n_kv, g.group, -1).sum(1)
        assert _ratio(bad, want).max() > ONE_ROW
        assert _ratio(got, want).max() <= ONE_ROW


@pytest.mark.parametrize("name,rows", [("B", 2), ("B", 40), ("R", 2), ("R", 40), ("R16", 200)])
def test_the_low_part_of_the_keys_is_added_first(name, rows):
    """What a chunk's scores lose on average, not at worst.  With the low part of K first the running sum is of full size only in
    the head_dim / 16 steps of the high part, over which it grows from nothing to X: half a dropped unit of 2^-23 a step is
    head_dim / 16 * X / 2 * 2^-24 * ln 2 = 2.6e-6 (128) or 5.3e-6 (256) of a weight with X = 2^4.  The normaliser loses the same of
    its keys, whose scores are about half as large: half of that is left.  (The high part first: one and a half times the dropped units
    more, 6e-6 measured at 256.)"""
    for g, got, want, _ in _weights(name, [16000], rows, 5):
        assert (_ratio(got, want) <= 3e-6).all(), _ratio(got, want).max()
