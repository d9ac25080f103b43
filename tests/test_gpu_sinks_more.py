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
