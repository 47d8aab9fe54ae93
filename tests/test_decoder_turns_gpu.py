"""DeviceDecoder over several turns: the limit of the cache."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def decoder(**options):
    from test_decoder_kv8_gpu import decoder
    return decoder("int4_gqa", **options)


def prompts(batch, n, seed=1):
    return np.random.default_rng(seed).integers(0, 700, (batch, n)).tolist()


def test_the_limit_counts_positions_that_a_caller_replayed(kt, oracle):
    """A caller that replays the captured step itself moves `length`; the checks of the cache's end follow it."""
    d = decoder(max_seq=16, kv_bits=8, kv_weights=True)
    d.prefill(prompts(1, 8))
    d.capture()
    for _ in range(8):
        d._graph.replay()
        d.length += 1
    assert d.held == 16
    with pytest.raises(ValueError):
        d.step(3)
    with pytest.raises(ValueError):
        d.prefill([[1]])
    d.evict(10, 2)
    assert d.held == 10 and d.length == 16 and d.cache.lengths.tolist() == [10]
    d.step(3)
    d.length += 5
    assert d.held == 16
    d.reset()
    assert d.held == d.length == 0
