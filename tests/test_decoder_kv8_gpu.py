"""DeviceDecoder with the 8-bit key/value cache, eviction and processed logits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

CONFIGS = {
    "int4_gqa": dict(vocab=1000, dim=256, layers=2, heads=4, kv_heads=2, hidden=512, rope_theta=500000.0,
                     rope_scaling=(8.0, 1.0, 4.0, 8192), bits=4, group_size=64, tied=False, qkv_bias=True),
    "int8_tied_mha": dict(vocab=768, dim=192, layers=2, heads=3, kv_heads=3, hidden=384, rope_theta=10000.0, bits=8,
                          group_size=64, tied=True, qkv_bias=False),
}
# A stored value is off by at most half a step of its block, 1/254 of the block's largest magnitude; through two
# layers of these models that moves the logits by less than a twentieth of their largest.
TOL = 0.05


def decoder(name, seed=7, **options):
    from kotensor_b200 import decoder as D
    from oracle import decoder_oracle as DO
    weights = DO.DecoderWeights.random(DO.DecoderConfig(**CONFIGS[name]), seed=seed)
    return D.DeviceDecoder(D.DecoderConfig(**CONFIGS[name]), weights, **options)


@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("block", [16, 64])
def test_logits_stay_near_the_fp32_cache(kt, oracle, name, block):
    a, b = decoder(name, max_seq=128), decoder(name, max_seq=128, kv_bits=8, kv_block=block)
    assert b.keys is None and b.cache.block == block
    prompt = np.random.default_rng(3).integers(0, 700, 37).tolist()
    for x, y in [(a.prefill(prompt), b.prefill(prompt))] + [(a.step(t), b.step(t)) for t in (5, 9, 300, 41)]:
        scale = x.abs().max()
        assert (x - y).abs().max() <= TOL * scale
    assert b.cache.lengths.tolist() == [41] and int(b.cache.status.item()) == 0
    # what the cache holds is the fp32 cache's rows, to half a step
    held = b.cache.k_codes[0, 0, :, :37].float() * b.cache.k_scales[0, 0].repeat_interleave(block, 1)[:, :37, None]
    want = a.keys[0, 0, :, :37]
    step = b.cache.k_scales[0, 0].repeat_interleave(block, 1)[:, :37, None]
    assert ((held - want).abs() <= 0.5001 * step + 1e-5 * want.abs().max()).all()


def test_a_batch_equals_its_sequences_and_replays(kt, oracle):
    prompts = np.random.default_rng(4).integers(0, 700, (3, 21)).tolist()
    batch = decoder("int4_gqa", max_seq=64, batch=3, kv_bits=8, kv_block=16)
    out = batch.generate_batch(prompts, 12)
    eager = decoder("int4_gqa", max_seq=64, batch=3, kv_bits=8, kv_block=16)
    eager.prefill(prompts)
    got = [eager.next_token.tolist()]
    for _ in range(11):
        eager.step(got[-1])
        got.append(eager.next_token.tolist())
    assert [list(r) for r in zip(*got)] == out  # replays of the captured step are the eager steps
    split = decoder("int4_gqa", max_seq=64, batch=3, kv_bits=8, kv_block=16)
    split.max_block_rows = 45  # two sequences to a block of the prefill
    assert torch.allclose(split.prefill(prompts), decoder("int4_gqa", max_seq=64, batch=3, kv_bits=8, kv_block=16).prefill(prompts),
                          atol=3e-2 * float(split.logits.abs().max()))


def test_generation_outgrows_the_cache(kt, oracle):
    prompts = np.random.default_rng(5).integers(0, 700, (2, 30)).tolist()
    d = decoder("int4_gqa", max_seq=48, batch=2, kv_bits=8, kv_block=16, kv_weights=True)
    out = d.generate_batch(prompts, 100, keep=24, recent=8)
    assert len(out[0]) == 100 and d.length == 30 + 99 and d.held <= 48
    assert d.cache.lengths.tolist() == [d.held, d.held] and int(d.cache.status.item()) == 0
    # every row and head gives away a weight of 1 a step, on what it keeps: nothing negative, nothing lost to NaN
    w = d.cache.weights[:, :, :, :d.held]
    assert bool((w >= 0).all()) and bool(w.isfinite().all())


def test_eviction_that_keeps_all_changes_nothing(kt, oracle):
    prompt = np.random.default_rng(6).integers(0, 700, 40).tolist()
    a = decoder("int8_tied_mha", max_seq=64, kv_bits=8, kv_weights=True)
    b = decoder("int8_tied_mha", max_seq=64, kv_bits=8, kv_weights=True)
    a.prefill(prompt)
    b.prefill(prompt)
    b.evict(40, 3)
    assert torch.equal(a.step(11), b.step(11))
    # the accumulated weights: each of the 41 rows and each head gave 1 in all
    total = a.cache.weights[:, 0, :, :41].double().sum(-1)
    assert bool(((total - 41).abs() < 1e-3).all())
    b.evict(20, 4)
    assert b.held == 20
    x = b.step(12)
    assert bool(x.isfinite().all()) and b.held == 21


def test_penalties_and_masks_steer_the_choice(kt, oracle):
    prompt = [[3, 4, 5], [6, 7, 8]]
    plain = decoder("int4_gqa", max_seq=64, batch=2)
    free = plain.generate_batch(prompt, 10)
    d = decoder("int4_gqa", max_seq=64, batch=2, kv_bits=8)
    d.penalize(presence=1e6)  # no token twice
    out = d.generate_batch(prompt, 30)
    for row in out:
        assert len(set(row)) == 30
    assert d._history[:, :5].tolist() == [p + o[:2] for p, o in zip(prompt, out)]
    d = decoder("int4_gqa", max_seq=64, batch=2, kv_bits=8)
    allowed = torch.zeros(2, 32, dtype=torch.int32, device="cuda")
    allowed[0, 1], allowed[1, 2] = 1 << 3, 1 << 5
    d.penalize(allowed=allowed)
    assert d.generate_batch(prompt, 4) == [[35] * 4, [69] * 4]
    # a bias on one token of the first sequence; without arguments the plain choice again
    fp32 = decoder("int4_gqa", max_seq=64, batch=2)
    fp32.penalize(bias_ids=torch.tensor([[77], [-1]], dtype=torch.int32, device="cuda"),
                  bias_values=torch.full((2, 1), 1e6, device="cuda"))
    biased = fp32.generate_batch(prompt, 10)
    assert biased[0] == [77] * 10 and biased[1] == free[1]
    fp32.reset()
    fp32.penalize()
    assert fp32.generate_batch(prompt, 10) == free


def test_refusals(kt, oracle):
    with pytest.raises(ValueError):
        decoder("int4_gqa", max_seq=64, kv_bits=4)
    with pytest.raises(ValueError):
        decoder("int4_gqa", max_seq=64, kv_weights=True)
    with pytest.raises(ValueError):
        decoder("int4_gqa", max_seq=64, kv_bits=8, kv_block=24)
    d = decoder("int4_gqa", max_seq=64, kv_bits=8)
    with pytest.raises(ValueError):
        d.evict(10, 2)
    with pytest.raises(ValueError):
        d.generate_batch([[1, 2]], 10, keep=5)
    with pytest.raises(ValueError):
        d.prefill(list(range(65)))
    w = decoder("int4_gqa", max_seq=64, kv_bits=8, kv_weights=True)
    for keep, recent in ((0, 0), (4, 5), (64, 1)):
        with pytest.raises(ValueError):
            w.generate_batch([[1, 2]], 10, keep=keep, recent=recent)
    with pytest.raises(ValueError):
        d.penalize(repetition=torch.ones(3))
    with pytest.raises(ValueError):
        d.cache.sequences(0, 2)
