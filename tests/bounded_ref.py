"""Plain 64-bit forms of the bounded-cache operators (sinks, accumulated weights, eviction) and the caches their tests use."""
from __future__ import annotations

import numpy as np
import torch

from tests.gpu_util import dev_i32, gpu_fill


def geom(name, **kw):
    from bruce_engine_b200.layout import F16, F32, G_B, G_R
    base = {"B": G_B, "B32": G_B.with_(out_dtype=F32), "R": G_R, "R16": G_R.with_(q_dtype=F16, out_dtype=F16),
            # one query head per kv head, and eight
            "B1": G_B.with_(n_head=4, n_kv=4), "B8": G_B.with_(n_head=16, n_kv=2)}[name]
    return base.with_(**kw)


def engine(g):
    from bruce_engine_b200.engine import AttnEngine
    return AttnEngine(g)


def values(rec: np.ndarray, hd: int) -> np.ndarray:
    """Records [..., record bytes] -> float64 [..., hd]: fp16 block scale times int8 value, exact."""
    nb = hd // 32
    d = np.ascontiguousarray(rec[..., :2 * nb]).view(np.float16).astype(np.float64)
    x = np.ascontiguousarray(rec[..., 2 * nb:]).view(np.int8).astype(np.float64)
    return x * np.repeat(d, 32, axis=-1)


def draw(g, n: int, rows: int, seed: int):
    """q [rows][n_head][hd] (as the geometry's q type holds it), k, v [n][n_kv][hd]; the first keys draw more attention."""
    rng = np.random.default_rng(seed)
    q = (1.5 * rng.standard_normal((rows, g.n_head, g.head_dim))).astype(np.float32)
    lean = rng.standard_normal((g.n_kv, g.head_dim))
    k = rng.standard_normal((n, g.n_kv, g.head_dim))
    k[:4] += lean
    q += 0.2 * np.repeat(lean, g.group, axis=0)
    # the tensor-core kernels take fp16 queries whatever type they come in
    return q.astype(np.float16).astype(np.float32), k.astype(np.float32), rng.standard_normal(
        (n, g.n_kv, g.head_dim)).astype(np.float32)


def quantised(g, k, v):
    """What the cache holds of k, v: records [n_kv][n][record], written by the library's own append."""
    n = k.shape[0] + (k.shape[0] & 1)
    e = engine(g.with_(slot_ctx=n, n_slots=1))
    kk, vv = e.alloc_kv_layer(False, fill=0)
    gpu_fill(e, k, v, kk, vv, False)
    torch.cuda.synchronize()
    return [t.cpu().numpy().reshape(g.n_kv, n, g.rec)[:, :k.shape[0]] for t in (kk, vv)]


def weights64(g, q, krec, p0: int, n_sink: int | None = None, window: int | None = None):
    """Softmax weights [n_head][rows][keys] in float64 (torch, on the GPU) of rows at p0 ...: causal, with `window` also windowed with sinks."""
    rows, n = q.shape[0], p0 + q.shape[0]
    kd = torch.from_numpy(values(krec[:, :n], g.head_dim)).cuda()
    qd = torch.from_numpy(q.astype(np.float64)).cuda().reshape(rows, g.n_kv, g.group, -1)
    scale = g.softmax_scale or g.head_dim ** -0.5
    a = torch.einsum("rhgd,hnd->hgrn", qd, kd).reshape(g.n_head, rows, n) * scale
    key, at = torch.arange(n, device="cuda")[None], (p0 + torch.arange(rows, device="cuda"))[:, None]
    see = key <= at
    if window is not None:
        see &= (key > at - window) | (key < n_sink)
    a = torch.where(see[None], a, -torch.inf)
    w = torch.exp(a - a.amax(-1, keepdim=True))
    return w / w.sum(-1, keepdim=True)


def attend64(g, q, krec, vrec, p0, n_sink=None, window=None):
    rows, n = q.shape[0], p0 + q.shape[0]
    w = weights64(g, q, krec, p0, n_sink, window).reshape(g.n_kv, g.group * rows, n)
    o = w @ torch.from_numpy(values(vrec[:, :n], g.head_dim)).cuda()
    return o.reshape(g.n_head, rows, -1).transpose(0, 1).cpu().numpy()


U = 2.0 ** -11        # half a step of fp16


def assert_attention(got, want, g, vrec, what=""):
    """An attention output against its value in 64 bits.

    Per element: the kernels form sum(p^ v^) / sum(p^) with p^ = p (1 + a), v^ = v (1 + b), |a|, |b| <= U, and round the
    result once more where the output is fp16.  The normalised weights then move by at most 2 U of themselves, the values by
    U, so  |got - want| <= (2 U + U) max|v_d| + U |want|, where v_d is the head's value at dimension d over all keys.  The
    scores add what fp32 leaves: a weight moves by at most |error of its exponent| ln 2, with exponents below 2^7 rounded to
    fp32 some four times (2^7 * 2^-24 * 4 = 2^-15), and the products of first order squared: half a U covers both.
    Per (row, head) and per row the 2-norm ratios are held to the tolerance of every attention path, 1e-3."""
    from tests.util import REL_TOL, errors
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want)
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    vmax = np.repeat(np.abs(values(vrec, g.head_dim)).max(1), g.group, axis=0)[None]           # [1][n_head][hd]
    tol = 3.5 * U * vmax + (U * np.abs(want) if g.out_dtype == 1 else 0.0)
    off = np.abs(got - want)
    assert (off <= tol).all(), f"{what}: {(off / np.maximum(tol, 1e-30)).max():.3f} of the bound per element"
    _, rel, _, relrow = errors(got, want)
    assert relrow <= REL_TOL and rel <= REL_TOL, f"{what}: relative per row {relrow:.3e}, per head {rel:.3e}"


class Paged:
    """Sequences of given records on scrambled pages; `skip(i, page)` leaves a page of sequence i unmapped."""

    def __init__(self, eng, recs, room: int, page_len: int, seed: int, skip=None, spare: int = 2):
        g = eng.geom
        rng = np.random.default_rng(seed)
        per = -(-max(r[0].shape[1] + room for r in recs) // page_len)
        need = [(i, p) for i, r in enumerate(recs) for p in range(-(-(r[0].shape[1] + room) // page_len))
                if skip is None or not skip(i, p)]
        self.n_pages = len(need) + spare
        order = rng.permutation(self.n_pages)
        self.table_np = np.full((len(recs), per), -1, dtype=np.int32)
        for j, (i, p) in enumerate(need):
            self.table_np[i, p] = order[j]
        self.table = torch.from_numpy(self.table_np).to(eng.device)
        self.desc, self.pk, self.pv = eng.alloc_pages(self.n_pages, page_len, self.table, fill=0x7F)
        for t, pool in ((0, self.pk), (1, self.pv)):
            host = pool.cpu().numpy().reshape(self.n_pages, g.n_kv, page_len, g.rec)
            for i, p in need:
                r = recs[i][t][:, p * page_len:(p + 1) * page_len]
                host[self.table_np[i, p], :, :r.shape[1]] = r
            pool.copy_(torch.from_numpy(host.reshape(-1)))
        self.page_len = page_len


def put(eng, buf, recs, is_swa: bool, which: int):
    """Records of every sequence into its partition of a contiguous layer buffer (a ring keeps the last 2 windows)."""
    g = eng.geom
    stride = g.pstride(is_swa)
    host = buf.cpu().numpy().reshape(g.n_slots, g.n_kv, stride, g.rec)
    for s, r in recs.items():
        x = r[which]
        n = x.shape[1]
        a = max(0, n - stride) if is_swa else 0
        host[s][:, np.arange(a, n) % stride] = x[:, a:]
    buf.copy_(torch.from_numpy(host.reshape(-1)))


def ids(x, eng):
    return dev_i32(x, eng.device)


def evict_list(score: np.ndarray, budget: int, n_sink: int, n_recent: int) -> np.ndarray:
    """Positions of one kv head that stay of len(score), ascending: NaN lowest, ties to the lower position."""
    n = len(score)
    if n <= budget:
        return np.arange(n)
    mid = np.arange(n_sink, n - n_recent)
    s = score[mid].astype(np.float64)
    order = np.lexsort((mid, np.where(np.isnan(s), 0.0, -s), np.isnan(s)))        # not NaN first, then best, then lowest
    keep = mid[order[:budget - n_sink - n_recent]]
    return np.concatenate([np.arange(n_sink), np.sort(keep), np.arange(n - n_recent, n)])


def score64(g, q, krec, p0: int, score_in):
    """Accumulated weights [n_kv][p0 + rows] in float64."""
    s = weights64(g, q, krec, p0).sum(1).reshape(g.n_kv, g.group, -1).sum(1).cpu().numpy()
    if score_in is not None:
        s[:, :p0] += score_in[:, :p0]
    return s


def assert_scores(got, want, g, q, krec, p0, what=""):
    """Accumulated weights against 64 bits.

    A weight is 2^(s - lse).  s is a sum of exact products in fp32 (blocks of 32 dims, then at most 8 scaled blocks): off by
    less than 16 * 2^-23 of A = sum |q_d k_d| * scale * log2(e), and so is lse, a convex mean of such errors; 2^x turns a
    difference d of exponents into a factor 1 + d ln 2.  The denominator adds n / 2 terms or fewer in a row, a position's
    weight at most rows * group: each addition is off by 2^-24 of a sum of positive terms.  ex2.approx is off by 2^-22, twice
    per weight and once per merge level: 8 * 2^-22.  The accumulated value adds one rounding."""
    n = krec.shape[1]
    kd = torch.from_numpy(values(krec, g.head_dim)).cuda().abs()
    qd = torch.from_numpy(q.astype(np.float64)).cuda().abs().reshape(q.shape[0], g.n_kv, g.group, -1)
    a = float(torch.einsum("rhgd,hnd->hgrn", qd, kd).max())
    a *= (g.softmax_scale or g.head_dim ** -0.5) * 1.4427
    rel = 2 * 0.6932 * 16 * 2.0 ** -23 * a + 8 * 2.0 ** -22 + (n / 2 + q.shape[0] * g.group) * 2.0 ** -24
    off = np.abs(np.asarray(got, dtype=np.float64) - want)
    tol = rel * np.abs(want) + 1e-30
    assert np.isfinite(got).all() and (off <= tol).all(), f"{what}: {np.nanmax(off / tol):.3f} of the bound ({rel:.2e})"
