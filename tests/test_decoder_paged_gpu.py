"""DeviceDecoder with the paged 16-bit key/value cache and drafted tokens."""
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
# A query, key, value or probability is off by at most half a step, 2^-8 of its size in bfloat16, as the 8-bit cache's
# are of their block's largest; through two layers of these models that moves the logits by less than a twentieth of
# their largest.  In float16 it is an eighth of that.
TOL = {torch.bfloat16: 0.05, torch.float16: 0.05 / 8}
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def no_wait_ran_out(kt):
    yield
    torch.cuda.synchronize()
    assert kt.Context.get(0).take_error() == 0


def decoder(name, seed=7, **options):
    from kotensor_b200 import decoder as D
    from oracle import decoder_oracle as DO
    weights = DO.DecoderWeights.random(DO.DecoderConfig(**CONFIGS[name]), seed=seed)
    return D.DeviceDecoder(D.DecoderConfig(**CONFIGS[name]), weights, **options)


@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("dtype,page", [(BF16, 64), (FP16, 16)])
def test_logits_stay_near_the_fp32_cache(kt, oracle, name, dtype, page):
    a, b = decoder(name, max_seq=128), decoder(name, max_seq=128, kv_bits=16, kv_page=page, kv_dtype=dtype)
    assert b.keys is None and b.cache.page == page
    prompt = np.random.default_rng(3).integers(0, 700, 37).tolist()
    for x, y in [(a.prefill(prompt), b.prefill(prompt))] + [(a.step(t), b.step(t)) for t in (5, 9, 300, 41)]:
        assert (x - y).abs().max() <= TOL[dtype] * x.abs().max()
    assert b.cache.lengths.tolist() == [41] and int(b.cache.status) == 0
    # what the cache holds are the fp32 cache's rows, rounded; the angles' products are exact here, off by up to
    # 41 * 2^-24 there
    pages = b.cache.table[0, :-(-41 // page)].long()
    for got, want in ((b.cache.keys, a.keys), (b.cache.values, a.values)):
        held = got[0, pages].transpose(0, 1).flatten(1, 2)[:, :41].float()
        want = want[0, 0, :, :41]
        assert ((held - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 1e-5 * want.abs().max()).all()


def test_a_batch_equals_its_sequences_and_replays(kt, oracle):
    prompts = np.random.default_rng(4).integers(0, 700, (3, 21)).tolist()
    options = dict(max_seq=64, batch=3, kv_bits=16, kv_page=16)
    out = decoder("int4_gqa", **options).generate_batch(prompts, 12)
    eager = decoder("int4_gqa", **options)
    eager.prefill(prompts)
    got = [eager.next_token.tolist()]
    for _ in range(11):
        eager.step(got[-1])
        got.append(eager.next_token.tolist())
    assert [list(r) for r in zip(*got)] == out  # replays of the captured step are the eager steps
    split = decoder("int4_gqa", **options)
    split.max_block_rows = 45  # two sequences to a block of the prefill
    assert torch.allclose(split.prefill(prompts), decoder("int4_gqa", **options).prefill(prompts),
                          atol=3e-2 * float(split.logits.abs().max()))


def test_pages_are_taken_as_the_texts_grow(kt, oracle):
    d = decoder("int4_gqa", max_seq=128, batch=2, kv_bits=16, kv_page=16, kv_pages=8)
    prompts = np.random.default_rng(5).integers(0, 700, (2, 20)).tolist()
    d.prefill(prompts)
    assert d.cache.free_pages == 4
    for i in range(12):
        d.step([1, 2])
    assert d.cache.free_pages == 4
    d.step([1, 2])
    assert d.cache.free_pages == 2 and d.length == 33
    with pytest.raises(ValueError, match="pages wanted"):
        d.prefill(np.random.default_rng(6).integers(0, 700, (2, 60)).tolist())
    assert d.length == 33
    d.reset()
    assert d.cache.lengths.tolist() == [0, 0]
    again = d.prefill(prompts).clone()
    assert torch.equal(again, decoder("int4_gqa", max_seq=128, batch=2, kv_bits=16, kv_page=16).prefill(prompts))


def chosen_by_the_model(name, prompts, texts, tol=0.1):
    """Every token of a text is the fp32 decoder's choice after those before it, up to logits that lie closer than
    the caches and the matmul kernels differ."""
    for prompt, text in zip(prompts, texts):
        d = decoder(name, max_seq=256)
        logits = d.prefill(prompt)
        for token in text:
            assert float(logits.max() - logits[token]) <= tol * float(logits.abs().max())
            logits = d.step(token)


@pytest.mark.parametrize("name,batch,nodes", [("int4_gqa", 1, 16), ("int4_gqa", 3, 5), ("int8_tied_mha", 2, 40), ("int4_gqa", 2, 1)])
def test_drafted_texts_are_the_models(kt, oracle, name, batch, nodes):
    prompts = np.random.default_rng(8).integers(0, 700, (batch, 19)).tolist()
    d = decoder(name, max_seq=160, batch=batch, kv_bits=16, kv_page=16)
    texts = d.generate_drafted(prompts, 60, nodes=nodes)
    assert [len(t) for t in texts] == [60] * batch and 1 <= d.passes <= 59
    if nodes == 1:
        assert d.passes == 59
    chosen_by_the_model(name, prompts, texts)
    # the sequences go on together
    assert d.cache.lengths.tolist() == [19 + 59] * batch and d.length == 78 and int(d.position) == 78
    assert d.next_token.tolist() == [t[-1] for t in texts]
    after = d.step([t[-1] for t in texts])
    whole = decoder(name, max_seq=160, batch=batch, kv_bits=16, kv_page=16)
    want = whole.prefill([p + t for p, t in zip(prompts, texts)])
    assert (after - want).abs().max() <= 0.1 * want.abs().max()
    # another call of the same decoder goes on from there
    more = d.generate_drafted([[3, 4]] * batch, 10, nodes=nodes)
    assert [len(t) for t in more] == [10] * batch and d.length == 79 + 2 + 9


def test_drafts_change_the_passes_and_not_the_text(kt, oracle):
    name, prompts = "int4_gqa", np.random.default_rng(9).integers(0, 700, (2, 12)).tolist()
    options = dict(max_seq=160, batch=2, kv_bits=16)
    truth = decoder(name, **options).generate_batch(prompts, 48)

    def told(text):  # the true continuation, behind a wrong one with the same beginning
        for p, t in zip(prompts, truth):
            if text[:12] == p and text[12:] == t[:len(text) - 12]:
                after = t[len(text) - 12:][:7]
                return [after[:2] + [999], after]
        return [[1, 2, 3]]

    d = decoder(name, **options)
    texts = d.generate_drafted(prompts, 48, nodes=12, draft=told)
    chosen_by_the_model(name, prompts, texts)
    passes = d.passes
    wrong = decoder(name, **options)
    worse = wrong.generate_drafted(prompts, 48, nodes=12, draft=lambda text: [[998, 997], [996]])
    chosen_by_the_model(name, prompts, worse)
    assert passes <= wrong.passes <= 47


def test_a_draft_that_fails_leaves_the_prompt(kt, oracle):
    prompts = np.random.default_rng(10).integers(0, 700, (2, 12)).tolist()
    d, e = (decoder("int4_gqa", max_seq=96, batch=2, kv_bits=16) for _ in range(2))

    def draft(text):
        if len(text) > 16:
            raise RuntimeError("no more")
        return [[7, 8]]

    with pytest.raises(RuntimeError, match="no more"):
        d.generate_drafted(prompts, 30, draft=draft)
    e.prefill(prompts)
    assert d.length == 12 and d.cache.lengths.tolist() == [12, 12] and d.next_token.tolist() == e.next_token.tolist()
    assert torch.equal(d.step([5, 6]), e.step([5, 6]))


def test_what_drafting_refuses(kt, oracle):
    prompts = [[1, 2, 3]]
    with pytest.raises(ValueError, match="kv_bits 16"):
        decoder("int4_gqa", max_seq=64).generate_drafted(prompts, 4)
    d = decoder("int4_gqa", max_seq=64, kv_bits=16)
    for nodes in (0, 1025):
        with pytest.raises(ValueError, match="nodes"):
            d.generate_drafted(prompts, 4, nodes=nodes)
    with pytest.raises(ValueError, match="max_tokens"):
        d.generate_drafted(prompts, 0)
    with pytest.raises(ValueError, match="exceed max_seq"):
        d.generate_drafted(prompts, 62)
    with pytest.raises(ValueError, match="eviction needs"):
        d.evict(4, 2)
    assert d.generate_drafted(prompts, 61, nodes=8) is not None  # to the last position
    d.reset()
    d.penalize(repetition=1.1)
    with pytest.raises(ValueError, match="penalties"):
        d.generate_drafted(prompts, 4)
    with pytest.raises(ValueError, match="kv_bits must be"):
        decoder("int4_gqa", max_seq=64, kv_bits=4)
