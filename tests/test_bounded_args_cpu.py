"""What the engine checks before a weight-accumulating call reaches the library, without a device: host tensors stand for the
device's, and a library that records the calls for libbattn."""
import types

import pytest
import torch

from bruce_engine_b200 import capi
from bruce_engine_b200.engine import AttnEngine
from bruce_engine_b200.layout import F16, Geom


class Elsewhere:
    """A scratch tensor of another device (or of the host)."""
    dtype, device, shape = torch.uint8, "elsewhere", (4096,)

    def get_device(self):
        return 7

    def is_contiguous(self):
        return True

    def numel(self):
        return 4096

    def element_size(self):
        return 1

    def data_ptr(self):
        return 4096


def _engine(calls):
    e = object.__new__(AttnEngine)
    e.geom = Geom(n_head=8, n_kv=2, slot_ctx=128, window=128, q_dtype=F16, out_dtype=F16)
    e.device = types.SimpleNamespace(index=torch.zeros(1).get_device())          # where host tensors are
    e.h, e.q_torch, e.out_torch = None, torch.float16, torch.float16
    e.lib = types.SimpleNamespace(battn_attend_track=lambda *a: calls.append(a) or 0,
                                  battn_attend_track_paged=lambda *a: calls.append(a) or 0)
    e._stream_here = lambda: 0
    return e


@pytest.mark.parametrize("paged", [False, True])
def test_the_scratch_of_an_accumulating_call_is_checked(paged):
    calls = []
    e = _engine(calls)
    g = e.geom
    q = torch.zeros(1, 1, g.n_head, g.head_dim, dtype=torch.float16)
    out, score, pos = torch.zeros_like(q), torch.zeros(1, g.n_kv, 128), torch.zeros(1, dtype=torch.int32)
    cache = [torch.zeros(g.n_kv * 128 * g.rec, dtype=torch.uint8) for _ in range(2)]

    def call(part):
        if paged:
            e.attn_track_paged(out, score, None, q, capi.CPages(0, 0, 0, 1, 1, 1, 128), pos, part)
        else:
            e.attn_track(out, score, None, q, *cache, pos, part)

    room = torch.zeros(4096, dtype=torch.uint8)
    for part, nbytes in ((room, 4096), (room.view(torch.float32), 4096), (room[256:], 3840)):
        call(part)
        a = calls.pop()
        ptr, size = a[-5:-3]                          # ..., ws, ws_bytes, rows, n_seq, stream
        assert (ptr, size) == (part.data_ptr(), nbytes)
    for part in (Elsewhere(), room[::2], room.view(64, 64)[:, :32]):
        with pytest.raises(ValueError, match="part"):
            call(part)
    assert not calls
