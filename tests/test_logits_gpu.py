"""kt_logits_process (kotensor_b200/logits.py) against oracle/kv8_oracle.py in 64
bits.  Tolerance: at most four float32 roundings of numbers no larger than
|x| * repetition + frequency * n + presence + sum |bias|, so 4 * 2^-24 of that."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def case(rows, vocab, history, biases, mask, seed=0, prompt=True):
    rng = np.random.default_rng(seed)
    a = {"logits": (3 * rng.standard_normal((rows, vocab))).astype(np.float32)}
    if history is not None:
        t = (vocab * rng.random((rows, max(1, history))) ** 3).astype(np.int32)
        t[rng.random(t.shape) < 0.02] = -1                    # padding
        t[rng.random(t.shape) < 0.02] = vocab
        a["tokens"] = t
        a["lengths"] = rng.integers(0, history + 1, rows).astype(np.int32)
        a["lengths"][0] = history
        if prompt:
            a["prompt_lengths"] = rng.integers(0, history + 1, rows).astype(np.int32)
        a["repetition"] = (1 + rng.random(rows)).astype(np.float32)
        a["frequency"] = rng.standard_normal(rows).astype(np.float32)
        a["presence"] = rng.standard_normal(rows).astype(np.float32)
    if biases:
        a["bias_ids"] = rng.integers(-1, vocab + 1, (rows, biases)).astype(np.int32)  # repeated ones among them
        a["bias_values"] = rng.standard_normal((rows, biases)).astype(np.float32)
        a["bias_counts"] = rng.integers(0, biases + 1, rows).astype(np.int32)
        a["bias_counts"][0] = biases
    if mask:
        a["allowed"] = rng.integers(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32)).astype(np.int32)
    return a


def bound(a):
    n = a["logits"].shape[1]
    size = np.abs(a["logits"]).astype(np.float64)
    for r in range(len(size)):
        if "repetition" in a:
            size[r] *= max(1.0, float(a["repetition"][r]))
        if "tokens" in a:
            line = a["tokens"][r, :max(0, int(a["lengths"][r]))]
            often = np.bincount(line[(line >= 0) & (line < n)], minlength=n)
            for key, times in (("frequency", often), ("presence", often > 0)):
                if key in a:
                    size[r] += abs(float(a[key][r])) * times
        if "bias_ids" in a:
            for i, x in zip(a["bias_ids"][r], a["bias_values"][r]):
                if 0 <= i < n:
                    size[r, i] += 2 * abs(float(x))
    return 4 * 2.0 ** -24 * size


def check(a, out, token):
    from oracle.kv8_oracle import process_logits
    want, best = process_logits(**a)
    got = out.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    assert (np.abs(got - np.where(fine, want, 0))[fine] <= bound(a)[fine]).all()
    for r, t in enumerate(token.tolist()):  # the greedy choice of what was written, the lowest index of equal ones
        line = np.where(np.isnan(got[r]), -np.inf, got[r])
        assert t == (int(line.argmax()) if line.max() > -1e9 else 0)


def run(kt, a, **more):
    from kotensor_b200.logits import LogitsProcessor
    rows, vocab = a["logits"].shape
    dev = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    p = LogitsProcessor(rows, vocab)
    out = torch.empty(rows, vocab, device="cuda")
    token = p(out=out, **{**dev, **more})
    again = torch.empty_like(out)
    second = p(out=again, **{**dev, **more}, next_token=torch.empty_like(token))
    assert torch.equal(out, again) and torch.equal(token, second)  # the scratch is left ready; equal bits
    return out, token, dev


@pytest.mark.parametrize("rows,vocab,history,biases,mask", [
    (1, 1, 0, 0, False),
    (1, 7, 3, 2, True),
    (2, 1000, 40, 0, False),
    (3, 1001, None, 5, True),        # rows that start off a 16-byte boundary
    (5, 8191, 300, 17, True),
    (4, 8192, 1, 0, True),
    (3, 8193, 2000, 300, False),
    (2, 32002, 100, 3, True),
    (1, 151936, 701, 20, False),
    (6, 128256, 513, 0, True),
])
def test_logits_match_64_bits(kt, rows, vocab, history, biases, mask):
    a = case(rows, vocab, history, biases, mask, seed=vocab)
    out, token, _ = run(kt, a)
    check(a, out, token)


@pytest.mark.parametrize("drop", [("repetition",), ("frequency", "presence"), ("presence", "prompt_lengths"),
                                  ("repetition", "frequency", "presence"), ("bias_counts",)])
def test_each_part_alone(kt, drop):
    a = {k: v for k, v in case(3, 5003, 200, 9, True, seed=5).items() if k not in drop}
    out, token, _ = run(kt, a)
    check(a, out, token)


def test_in_place_and_strided_rows(kt):
    """Logits inside a wider buffer, processed where they are; an output of another alignment."""
    from kotensor_b200.logits import LogitsProcessor
    a = case(3, 9001, 100, 4, True, seed=9)
    dev = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    p = LogitsProcessor(3, 9001)
    wide = torch.full((3, 9100), 7.0, device="cuda")
    wide[:, 5:9006] = dev["logits"]
    token = p(wide[:, 5:9006], **{k: v for k, v in dev.items() if k != "logits"})
    check(a, wide[:, 5:9006], token)
    assert bool((wide[:, :5] == 7).all()) and bool((wide[:, 9006:] == 7).all())
    other = torch.full((3, 9100), 7.0, device="cuda")
    p(dev["logits"], out=other[:, 2:9003], **{k: v for k, v in dev.items() if k != "logits"})
    assert torch.equal(other[:, 2:9003], wide[:, 5:9006])
    assert bool((other[:, :2] == 7).all()) and bool((other[:, 9003:] == 7).all())


def test_shared_lists(kt):
    """One token list, bias list and mask for all rows (stride 0)."""
    a = case(4, 3000, 50, 6, True, seed=11)
    for k in ("tokens", "bias_ids", "bias_values", "allowed"):
        a[k][:] = a[k][:1]
    from kotensor_b200.logits import LogitsProcessor
    dev = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    for k in ("tokens", "bias_ids", "bias_values", "allowed"):
        dev[k] = dev[k][:1].expand(4, -1)
    out = torch.empty(4, 3000, device="cuda")
    token = LogitsProcessor(4, 3000)(out=out, **dev)
    check(a, out, token)


def test_rows_with_nothing_to_choose(kt):
    """All forbidden, all NaN, all at or below -1e9: token 0; ties: the lowest index; -0 and 0 are equal."""
    from kotensor_b200.logits import LogitsProcessor
    n = 20000
    x = torch.randn(7, n, device="cuda")
    allowed = torch.full((7, 625), -1, dtype=torch.int32, device="cuda")
    allowed[0] = 0
    x[1] = float("nan")
    x[2] = -1e9
    x[3] = float("-inf")
    x[4].clamp_(max=2.0)
    x[4, 19000:19010] = 2.0
    x[4, 12345] = 2.0
    x[5] = -1.0
    x[5, 17000] = -0.0
    x[5, 18000] = 0.0
    x[6, 9] = float("nan")
    x[6, 15000] = float("inf")
    before = x.clone()
    token = LogitsProcessor(7, n)(x, allowed=allowed).tolist()
    assert token[:4] == [0, 0, 0, 0]
    assert token[4] == int((before[4] == 2.0).nonzero()[0]) and token[5] == 17000 and token[6] == 15000
    assert bool(x[0].isneginf().all()) and torch.equal(x[4:].nan_to_num(), before[4:].nan_to_num())


def test_refusals(kt):
    from kotensor_b200.logits import LogitsProcessor
    with pytest.raises(ValueError):
        LogitsProcessor(0, 5)
    p = LogitsProcessor(2, 100)
    x = torch.zeros(2, 100, device="cuda")
    one, ids = torch.ones(2, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    for bad in (dict(logits=x[:1]), dict(logits=x.double()), dict(logits=x.cpu()), dict(logits=x, tokens=ids),
                dict(logits=x, repetition=one), dict(logits=x, bias_ids=ids),
                dict(logits=x, bias_ids=ids, bias_values=torch.zeros(2, 4, device="cuda")),
                dict(logits=x, tokens=ids.long(), lengths=n), dict(logits=x, tokens=ids, lengths=n[:1]),
                dict(logits=x, allowed=torch.zeros(2, 3, dtype=torch.int32, device="cuda")),
                dict(logits=x, out=x[:, :50]), dict(logits=x.t().contiguous().t())):
        with pytest.raises(ValueError):
            p(**bad)
    with pytest.raises(ValueError):
        LogitsProcessor(1, 100)(x[:1], repetition=one[:1])
