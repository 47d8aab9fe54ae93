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


# Only the 8-bit cache drops tokens past its end; what the fp32 cache does there is refused before a launch.
@pytest.mark.parametrize("bits", [8, 32])
def test_a_second_turn_that_does_not_fit_is_refused(kt, oracle, bits):
    d = decoder(max_seq=48, batch=2, kv_bits=bits)
    first = d.generate_batch(prompts(2, 10), 12)          # 21 positions
    assert d.held == d.length == 21
    with pytest.raises(ValueError):
        d.generate_batch(prompts(2, 10, seed=2), 19)      # 21 + 10 + 18 = 49
    assert d.held == 21 and int(d.position.item()) == 21  # refused before anything ran
    second = d.generate_batch(prompts(2, 10, seed=2), 18)  # 48: the last position is used
    assert d.held == 48 and all(len(x) == 18 for x in second) and len(first[0]) == 12
    one = decoder(max_seq=32, kv_bits=bits)
    one.generate(prompts(1, 6)[0], 10)
    assert one.held == 15
    with pytest.raises(ValueError):
        one.generate(prompts(1, 6)[0], 13)
    assert one.held == 15
    one.generate(prompts(1, 6)[0], 12)
    assert one.held == 32
    with pytest.raises(ValueError):
        one.step(3)


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


def test_dropped_tokens_are_an_error(kt, oracle):
    """A cache that holds more than the decoder knows: the tokens it drops end the generation with an error."""
    d = decoder(max_seq=32, batch=2, kv_bits=8)
    d.cache.lengths.fill_(d.cache.capacity - 5)
    with pytest.raises(ValueError):
        d.generate_batch(prompts(2, 4), 10)
    d.reset()
    assert len(d.generate_batch(prompts(2, 4), 10)[0]) == 10
