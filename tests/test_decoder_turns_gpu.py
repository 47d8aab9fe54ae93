"""DeviceDecoder over several turns: the cache's limit, the tokens that penalties
remember, and penalties that change in the middle of a text."""
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


def repeats(tokens, window):
    return [i for i, t in enumerate(tokens) if t in tokens[max(0, i - window):i]]


def test_penalties_hold_past_the_history(kt, oracle):
    """With a history of n tokens, no token comes again within n: long past the cache's end, for texts whose
    prompt is shorter and longer than the history, and over a second prompt."""
    for history, n in ((None, 20), (16, 5), (16, 30), (7, 7), (1, 3)):
        d = decoder(max_seq=48, batch=2, kv_bits=8, kv_block=16, kv_weights=True)
        d.penalize(presence=1e6, repetition=None, history=history)
        text = prompts(2, n, seed=n)
        for turn in range(2):
            out = d.generate_batch(text, 120, keep=24, recent=8)
            for q in range(2):
                assert repeats(out[q], history or 48) == [], (history, n, turn)
            text = prompts(2, 4, seed=turn)
            d.evict(24, 8)


def remembered(text, split, room):
    """What penalties see of `text`, of which the first `split` are the prompt: (tokens in any order, answer's)."""
    last = text[-room:]
    cut = max(0, split - (len(text) - len(last)))
    return sorted(last), sorted(last[cut:])


def seen(d, q=0):
    n, p = int(d._history_lengths[q].item()), int(d._prompt_lengths[q].item())
    line = [t for t in d._history[q, :n].tolist()]
    return sorted(t for t in line if t >= 0), sorted(t for t in line[max(0, p):] if t >= 0)


@pytest.mark.parametrize("room,first", [(5, 3), (5, 5), (5, 9), (1, 1), (8, 1), (40, 4)])
def test_the_history_is_the_last_tokens(kt, oracle, room, first):
    """Token by token against a list, over prompts, steps, a second prompt and more steps."""
    d = decoder(max_seq=200, kv_bits=8)
    d.penalize(frequency=0.5, history=room)
    rng = np.random.default_rng(room)
    text, split = [], 0
    for n in (first, 4, 1):
        part = rng.integers(0, 700, n).tolist()
        d.prefill([part])
        text += part
        split = len(text)  # all that is there when a prompt comes counts as prompt
        assert seen(d) == remembered(text, split, room)
        for _ in range(3 * room + 2 if room < 10 else 12):
            t = int(rng.integers(0, 700))
            d.step(t)
            text.append(t)
            assert seen(d) == remembered(text, split, room)


def test_penalties_in_the_middle_of_a_text(kt, oracle):
    """`penalize` after a prompt and some answer counts what has been processed; again, it changes the penalties
    and keeps what is remembered; taken back and given again, nothing is lost."""
    text = prompts(2, 6)
    early, late = (decoder(max_seq=200, batch=2, kv_bits=8) for _ in range(2))
    early.penalize(presence=0.0)
    a, b = early.generate_batch(text, 10), late.generate_batch(text, 10)
    assert a == b
    for d in (early, late):
        d.penalize(presence=1e6)
    for q in range(2):
        want = remembered(text[q] + a[q][:-1], 6, 200)
        assert seen(early, q) == want and seen(late, q) == want
    for d in (early, late):
        for _ in range(5):
            d.step(d.next_token.tolist())
    x = early.next_token.tolist()
    assert x == late.next_token.tolist()
    for q in range(2):
        assert x[q] not in a[q][:-1]
    late.penalize()
    late.step(x)
    late.penalize(presence=1e6)
    early.step(x)
    for q in range(2):
        assert seen(late, q) == seen(early, q)
    late.penalize(presence=1e6, history=4)
    assert len(seen(late)[0]) == 4 and set(seen(late)[0]) <= set(seen(early)[0])
    # generate, one sequence: prompt tokens count as prompt
    one = decoder(max_seq=64, kv_bits=8)
    out = one.generate(text[0], 8)
    one.penalize(repetition=1.5)
    assert seen(one) == remembered(text[0] + out[:-1], 6, 64)
    one.reset()
    assert seen(one) == ([], [])
    one.generate(text[1], 4)
    one.penalize(repetition=1.25)
    assert seen(one)[0] == sorted(text[1] + one_answer(one, text[1], 4))


def one_answer(d, prompt, n):
    """The first n - 1 tokens that follow `prompt` under repetition 1.5, on a fresh decoder."""
    e = decoder(max_seq=64, kv_bits=8)
    e.penalize(repetition=1.5)
    return e.generate(prompt, n)[:-1]
