"""What the engine checks before a call of the bounded caches reaches the library, without a device: host tensors stand for the
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


def _engine(calls, n_slots=1):
    e = object.__new__(AttnEngine)
    e.geom = Geom(n_head=8, n_kv=2, slot_ctx=128, window=128, n_slots=n_slots, q_dtype=F16, out_dtype=F16)
    e.device = types.SimpleNamespace(index=torch.zeros(1).get_device())          # where host tensors are
    e.h, e.q_torch, e.out_torch = None, torch.float16, torch.float16
    e._ws_need = {(1, 1): 256}
    e.lib = types.SimpleNamespace(**{name: lambda *a: calls.append(a) or 0 for name in (
        "battn_attend_track", "battn_attend_track_paged", "battn_attend_sinks", "battn_sinks_store")})
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


def test_slots_are_named_over_sink_buffers_of_all_slots():
    calls = []
    e = _engine(calls, n_slots=3)
    g = e.geom
    q = torch.zeros(1, 1, g.n_head, g.head_dim, dtype=torch.float16)
    ring = [torch.zeros(3 * g.n_kv * 256 * g.rec, dtype=torch.uint8) for _ in range(2)]
    k, v = (torch.zeros(3, g.n_kv * 128 * g.rec, dtype=torch.uint8) for _ in range(2))
    pos, slot, part = torch.zeros(1, dtype=torch.int32), torch.full((1,), 2, dtype=torch.int32), torch.zeros(256, dtype=torch.uint8)

    def attend(sinks, kslot):
        e.attn_sinks(torch.zeros_like(q), q, *ring, sinks, pos, part, kslot=kslot)
        e.sinks_store(*ring, sinks, pos, kslot=kslot)

    for sinks, kslot in ((e.sinks(4, k, v), slot), (e.sinks(4, k, v, cap=128), slot), (e.sinks(4, k[2], v[2], cap=128), None),
                         (e.sinks(4, k, v), None), (capi.CSinks(k.data_ptr(), v.data_ptr(), 4, 128), slot)):
        attend(sinks, kslot)
        assert len(calls) == 2
        calls.clear()
    one = e.sinks(4, k[2], v[2], cap=128)
    for f in (lambda: e.attn_sinks(torch.zeros_like(q), q, *ring, one, pos, part, kslot=slot),
              lambda: e.sinks_store(*ring, one, pos, kslot=slot)):
        with pytest.raises(ValueError, match="slots"):
            f()
    assert not calls
