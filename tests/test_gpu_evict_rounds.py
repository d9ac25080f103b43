"""Evictions whose move takes several rounds of two buffers, the next round's loads over this round's stores: batches that have
more clusters of eight CTAs than the SMs hold at one CTA each, with budgets above eight rounds of 256 records (head_dim 128) or
128 (256).  Every byte is compared with the plain form, as in test_gpu_evict."""
import pytest

from tests.test_gpu_evict import _case

pytestmark = pytest.mark.gpu

# sequences, budget: three rounds with a partial, odd last one; exactly two full rounds; one record into the second round
SHAPES = {"B": (([7001, 6000, 2500], 5001), ([4500, 4097, 9000], 4096), ([2600, 2100, 2049, 3001], 2049)),
          "R": (([3100, 2600, 2501, 900], 2500), ([2300, 2049, 4000, 2050], 2048), ([1100, 1500, 1026, 2000], 1025))}


@pytest.mark.parametrize("store", ["slots", "paged"])
@pytest.mark.parametrize("to_other", [False, True])
@pytest.mark.parametrize("name", ["B", "R"])
def test_rounds_of_two_buffers(name, to_other, store):
    for j, (lens, budget) in enumerate(SHAPES[name]):
        for kind, n_sink, n_recent in (("weights", 4, 100), ("ties", 0, 0), ("weights", budget // 2, 1)):
            _case(name, lens, budget, n_sink, n_recent, store, kind, to_other=to_other, seed=j)


def test_rounds_beside_idle_sequences():
    for store in ("slots", "paged"):
        _case("B", [7001, 6000, 5500, 2500], 5001, 4, 100, store, act=[1, 0, 1, 1], seed=9)
        _case("R", [3100, 2600, 4000, 900, 3001], 2500, 0, 0, store, "odd", to_other=True, act=[0, 1, 1, 1, 0], seed=9)
