"""The 8-bit key/value cache (kotensor_b200/kv8.py) against oracle/kv8_oracle.py:
what is stored and evicted bit for bit, attention and accumulated weights within
the rounding of fp32 sums.

Attention tolerance: a score of magnitude-sum S = sum |scale q k| carries an fp32
rounding error of about sqrt(d) 2^-24 S; four times that, plus 2^-20 for the
exponential and the sums of the softmax, bounds the relative error of every
weight, and times max |v| the error of the context."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def make(kt, b, h, d, capacity, block, lengths, seed=0, fill=True, layers=1):
    """A device cache and its oracle holding the same random tokens; slots that hold
    nothing have codes of all values and scales that are not finite."""
    from kotensor_b200.kv8 import KVCache8
    from oracle.kv8_oracle import Cache
    cache = KVCache8(layers, b, h, d, capacity, block, track_weights=True)
    ref = Cache(b, h, d, cache.capacity, block, [0] * b)
    rng = np.random.default_rng(seed)
    for n in "kv":
        ref.codes[n][:] = rng.integers(-128, 128, ref.codes[n].shape)
        ref.scales[n][:] = rng.choice(np.array([np.nan, np.inf, -np.inf], np.float32), ref.scales[n].shape)
        ref.tail[n][:] = np.nan
    ref.weights[:] = np.nan
    if fill and max(lengths) > 0:
        rows = max(lengths)
        k = rng.standard_normal((b * rows, h * d), dtype=np.float32) * np.exp(rng.standard_normal(h * d)).astype(np.float32)
        v = rng.standard_normal((b * rows, h * d), dtype=np.float32)
        ref.store(k, v, rows, lengths)
    ref.lengths[:] = lengths
    push(cache, ref)
    return cache, ref, rng


def push(cache, ref, layer=0):
    for n in "kv":
        getattr(cache, n + "_codes")[layer].copy_(torch.from_numpy(ref.codes[n]))
        getattr(cache, n + "_scales")[layer].copy_(torch.from_numpy(ref.scales[n]))
        getattr(cache, n + "_tail")[layer].copy_(torch.from_numpy(ref.tail[n]))
    cache.weights[layer].copy_(torch.from_numpy(ref.weights))
    cache.lengths.copy_(torch.from_numpy(ref.lengths))


def assert_same(cache, ref, layer=0):
    for n in "kv":
        for what in ("codes", "scales", "tail"):
            got = getattr(cache, f"{n}_{what}")[layer].cpu().numpy()
            want = getattr(ref, what)[n]
            assert np.array_equal(got, want, equal_nan=what != "codes"), (n, what)
    assert np.array_equal(cache.weights[layer].cpu().numpy(), ref.weights, equal_nan=True)


@pytest.mark.parametrize("b,h,d,block,lengths,rows", [
    (1, 1, 16, 16, [0], 1),
    (1, 2, 64, 64, [63], 1),            # the token that fills a block
    (3, 2, 48, 16, [0, 15, 16], 1),
    (2, 3, 128, 32, [31, 40], 2),
    (2, 1, 80, 64, [5, 127], 70),
    (4, 2, 96, 16, [0, 1, 17, 100], 33),
    (1, 8, 128, 64, [1], 129),
])
def test_store_is_the_defined_quantisation(kt, b, h, d, block, lengths, rows):
    cache, ref, rng = make(kt, b, h, d, 256, block, lengths, seed=rows)
    k = rng.standard_normal((b * rows, h * d), dtype=np.float32) * np.float32(3.0)
    v = rng.standard_normal((b * rows, h * d), dtype=np.float32) * np.float32(1e-3)
    ref.store(k, v, rows)
    cache.store(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), rows)
    assert_same(cache, ref)
    assert int(cache.status.item()) == 0
    # in 64 bits: every value held is the nearest multiple of its scale to the value given
    for n, x in (("k", k), ("v", v)):
        x = x.reshape(b, rows, h, d).astype(np.float64)
        for i in range(b):
            for j in range(h):
                held = cache_values(cache, n, i, j)[lengths[i]:lengths[i] + rows]
                step = np.repeat(ref.scales[n][i, j], block)[lengths[i]:lengths[i] + rows, None]
                # half a step, and five float32 roundings (1/a, 127/a, x * inverse, 1/127, scale) of at most 127 steps
                assert (np.abs(held - x[i, :, j]) <= step * (0.5 + 127 * 5 * 2.0 ** -24)).all()


def cache_values(cache, name, b, h, layer=0):
    codes = getattr(cache, name + "_codes")[layer, b, h].cpu().numpy().astype(np.float64)
    scales = getattr(cache, name + "_scales")[layer, b, h].cpu().numpy().astype(np.float64)
    return codes * np.repeat(scales, cache.block)[:, None]


def test_store_does_not_depend_on_the_split_into_calls(kt):
    whole, ref, rng = make(kt, 2, 2, 64, 256, 32, [7, 32])
    parts, _, _ = make(kt, 2, 2, 64, 256, 32, [7, 32])
    rows = 90
    k = torch.from_numpy(rng.standard_normal((2, rows, 128), dtype=np.float32)).cuda()
    v = torch.from_numpy(rng.standard_normal((2, rows, 128), dtype=np.float32)).cuda()
    whole.store(0, k.reshape(-1, 128), v.reshape(-1, 128), rows)
    whole.advance(rows)
    at = 0
    for n in (1, 1, 30, 2, 55, 1):
        parts.store(0, k[:, at:at + n].reshape(-1, 128), v[:, at:at + n].reshape(-1, 128), n)
        parts.advance(n)
        at += n
    assert at == rows
    assert torch.equal(whole.lengths, parts.lengths)
    for b, n in enumerate(whole.lengths.tolist()):
        for x in "kv":
            assert torch.equal(getattr(whole, x + "_codes")[0, b, :, :n], getattr(parts, x + "_codes")[0, b, :, :n])
            assert torch.equal(getattr(whole, x + "_scales")[0, b, :, :-(-n // 32)],
                               getattr(parts, x + "_scales")[0, b, :, :-(-n // 32)])
            assert torch.equal(getattr(whole, x + "_tail")[0, b, :, :n % 32], getattr(parts, x + "_tail")[0, b, :, :n % 32])


def test_store_counts_and_capacity(kt):
    """Rows past counts[b] are not tokens; tokens past the capacity are dropped and reported."""
    cache, ref, rng = make(kt, 5, 2, 32, 64, 16, [0, 10, 33, 60, 64])
    counts = np.array([0, 3, 40, -2, 1], np.int32)
    k = rng.standard_normal((5 * 7, 64), dtype=np.float32)
    assert not ref.store(k, k, 7, [0, 3, 7, 0, 0])
    cache.store(0, torch.from_numpy(k).cuda(), torch.from_numpy(k).cuda(), 7,
                counts=torch.from_numpy(np.array([0, 3, 40, -2, 0], np.int32)).cuda())
    assert_same(cache, ref)
    assert int(cache.status.item()) == 0
    assert ref.store(k, k, 7, counts)
    cache.store(0, torch.from_numpy(k).cuda(), torch.from_numpy(k).cuda(), 7, counts=torch.from_numpy(counts).cuda())
    assert_same(cache, ref)
    assert int(cache.status.item()) == 1


@pytest.mark.parametrize("offset,stride_extra", [(0, 4), (1, 0), (2, 3), (4, 64)])
def test_store_from_strided_unaligned_rows(kt, offset, stride_extra):
    cache, ref, rng = make(kt, 2, 2, 48, 128, 16, [3, 20])
    rows, width = 5, 96
    base = torch.from_numpy(rng.standard_normal(offset + 10 * (2 * width + stride_extra) + 8, dtype=np.float32)).cuda()
    both = base[offset:offset + 10 * (2 * width + stride_extra)].reshape(10, 2 * width + stride_extra)
    k, v = both[:, :width], both[:, width:2 * width]
    ref.store(k.cpu().numpy(), v.cpu().numpy(), rows)
    cache.store(0, k, v, rows)
    assert_same(cache, ref)


def test_store_of_values_that_are_not_ordinary(kt):
    """Zeros, values below 2^-100, the largest floats, and NaN / infinity in one block of several."""
    cache, ref, rng = make(kt, 1, 6, 16, 64, 16, [0])
    x = np.zeros((32, 6, 16), np.float32)
    x[:, 0] = 0.0
    x[:, 1] = 2.0 ** -101
    x[:, 2] = rng.standard_normal((32, 16)) * 1e-29
    x[:, 3] = rng.choice([3.4e38, -3.4e38, 1e38], (32, 16))
    x[:, 4] = rng.standard_normal((32, 16))
    x[5, 4, 3] = np.nan
    x[:, 5] = rng.standard_normal((32, 16))
    x[20, 5, 0] = -np.inf
    x = x.reshape(32, 96)
    ref.store(x, x, 32)
    cache.store(0, torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda(), 32)
    assert_same(cache, ref)
    assert np.isnan(ref.scales["k"][0, 4, 0]) and np.isfinite(ref.scales["k"][0, 4, 1])
    assert np.isnan(ref.scales["k"][0, 5, 1]) and np.isfinite(ref.scales["k"][0, 5, 0])


def attention_case(kt, b, heads, h, d, block, lengths, rows, counts=None, seed=1, scale=None, capacity=None, gain=1.0):
    capacity = capacity or max(lengths) + rows + 3
    cache, ref, rng = make(kt, b, h, d, capacity, block, lengths, seed=seed)
    k = rng.standard_normal((b * rows, h * d), dtype=np.float32)
    v = rng.standard_normal((b * rows, h * d), dtype=np.float32)
    ref.store(k, v, rows, counts)
    push(cache, ref)
    q = (gain * rng.standard_normal((b * rows, heads * d))).astype(np.float32)
    c = None if counts is None else torch.from_numpy(np.array(counts, np.int32)).cuda()
    got = cache.attend(0, torch.from_numpy(q).cuda(), heads, rows, scale=scale, counts=c, accumulate=True)
    want, weights, size, top = ref.attend(q, heads, rows, scale if scale is not None else d ** -0.5, counts)
    near = 4 * d ** 0.5 * 2.0 ** -24 * size + 2.0 ** -20
    err = np.abs(got.cpu().numpy() - want).max(initial=0)
    assert np.isfinite(got.cpu().numpy()).all()
    assert err <= near * top, (err / max(top, 1e-30), near)
    after = cache.weights[0].cpu().numpy().astype(np.float64)
    for i in range(b):
        m = rows if counts is None else max(0, min(rows, counts[i]))
        n = min(lengths[i] + m, cache.capacity)
        before = ref.weights[i, :, :n].astype(np.float64)
        total = weights[i, :, :n]
        assert (np.abs(after[i, :, :n] - before - total) <= near * total + 2.0 ** -23 * (before + total) + 1e-30).all()
        # slots that hold nothing are left alone
        assert np.array_equal(after[i, :, n:], ref.weights[i, :, n:].astype(np.float64), equal_nan=True)
    # without the weights: the same context, bit for bit
    kept = cache.weights.clone()
    again = cache.attend(0, torch.from_numpy(q).cuda(), heads, rows, scale=scale, counts=c)
    assert torch.equal(again, got)
    assert torch.equal(cache.weights.isnan(), kept.isnan()) and torch.equal(cache.weights.nan_to_num(), kept.nan_to_num())
    return cache, ref


@pytest.mark.parametrize("b,heads,h,d,block,lengths", [
    (1, 1, 1, 16, 16, [0]),                       # one token, one head
    (1, 14, 2, 64, 64, [300]),
    (2, 7, 7, 64, 16, [1, 64]),
    (3, 32, 8, 128, 64, [0, 63, 200]),
    (2, 15, 5, 80, 32, [31, 33]),
    (2, 24, 2, 96, 16, [15, 129]),                # 12 heads to a group
    (1, 40, 2, 48, 32, [77]),                     # 20 heads to a group
    (5, 8, 1, 112, 64, [0, 1, 500, 64, 1000]),    # ragged
    (1, 32, 8, 128, 64, [4095]),
    (1, 8, 1, 128, 16, [20011]),                  # long, one key head
    (40, 4, 2, 32, 32, list(range(0, 200, 5))),
])
def test_attention_of_one_row(kt, b, heads, h, d, block, lengths):
    attention_case(kt, b, heads, h, d, block, lengths, 1, seed=heads)


@pytest.mark.parametrize("b,heads,h,d,block,lengths,rows", [
    (1, 1, 1, 16, 16, [0], 2),
    (2, 4, 2, 64, 64, [0, 100], 3),
    (1, 32, 8, 128, 64, [130], 17),
    (2, 14, 2, 64, 32, [1, 250], 65),
    (1, 15, 5, 80, 16, [0], 129),
    (3, 12, 1, 96, 64, [64, 7, 0], 31),
    (1, 8, 2, 128, 64, [1000], 200),
    (2, 6, 6, 112, 32, [3, 90], 130),
    (2, 8, 2, 128, 64, [5000, 3], 70),            # slots split between CTAs, one sequence with fewer than splits
    (1, 14, 2, 64, 16, [3000], 90),
    (3, 32, 8, 64, 32, [700, 0, 64], 33),
])
def test_attention_of_several_rows(kt, b, heads, h, d, block, lengths, rows):
    attention_case(kt, b, heads, h, d, block, lengths, rows, seed=rows)


@pytest.mark.parametrize("b,heads,h,d,block,lengths,rows", [
    (2, 28, 4, 80, 16, [700, 3], 150),            # a group of 7, slots of several CTAs, vectors shared by a cluster
    (1, 7, 1, 128, 64, [20], 600),                # slots that only later rows see
    (1, 16, 16, 48, 32, [300], 140),
])
def test_weights_of_many_rows(kt, b, heads, h, d, block, lengths, rows):
    """Weights of prompts, twice with equal bits, and from queries at any address."""
    cache, ref = attention_case(kt, b, heads, h, d, block, lengths, rows, seed=d)
    room = torch.randn(b * rows * (heads * d + 3) + 1, device="cuda")
    shifted = room[1:].reshape(b * rows, heads * d + 3)[:, :heads * d]
    results = []
    for q in (shifted, shifted.contiguous(), shifted):
        cache.weights.zero_()
        context = cache.attend(0, q, heads, rows, accumulate=True)
        results.append((context, cache.weights.clone()))
    for context, weights in results[1:]:
        assert torch.equal(context, results[0][0]) and torch.equal(weights, results[0][1])
    # every row hands out one unit of weight per query head; each exponential's relative error is below 2^-16
    given = results[0][1].double().sum() / (b * rows * heads)
    assert abs(float(given) - 1.0) < 2.0 ** -16


@pytest.mark.parametrize("rows", [1, 5, 20, 70])
def test_attention_counts(kt, rows):
    """Rows past counts[b] give zeros and no weights; a sequence may have none at all."""
    lengths, counts = [0, 9, 120, 33], [0, rows, rows - 1, 1]
    cache, ref = attention_case(kt, 4, 8, 2, 64, 32, lengths, rows, counts=counts)
    out = cache.attend(0, torch.randn(4 * rows, 512, device="cuda"), 8, rows,
                       counts=torch.tensor(counts, dtype=torch.int32, device="cuda")).reshape(4, rows, 512)
    for b, n in enumerate(counts):
        assert bool((out[b, n:] == 0).all()) and (n == 0 or bool((out[b, :n] != 0).any()))


def test_attention_of_scores_far_apart(kt):
    """Large queries: the softmax is nearly one slot's, and its exponents span hundreds."""
    attention_case(kt, 2, 8, 2, 64, 16, [40, 300], 1, gain=50.0)
    attention_case(kt, 1, 8, 2, 64, 16, [100], 20, gain=50.0)


def test_attention_of_small_and_large_magnitudes(kt):
    """Scales of key and value blocks over many orders of magnitude: no fixed-point step loses the small ones."""
    for rows in (1, 12):
        cache, ref, rng = make(kt, 1, 2, 64, 512, 16, [400 - rows])
        for n, low in (("k", 1e-4), ("v", 1e-12)):
            x = rng.standard_normal((400, 2, 64)).astype(np.float32)
            x[:, 0] *= np.exp(rng.uniform(np.log(low), 0, (25, 1, 1))).repeat(16, 0)[:, 0].astype(np.float32)
            x[:, 1] *= np.float32(1e-20 if n == "v" else 1.0)
            for h in range(2):
                for i in range(25):
                    from oracle.kv8_oracle import quantise
                    ref.codes[n][0, h, 16 * i:16 * i + 16], ref.scales[n][0, h, i] = quantise(x[16 * i:16 * i + 16, h])
        push(cache, ref)
        q = (1e6 * rng.standard_normal((rows, 128))).astype(np.float32)
        scale = 1e-6
        got = cache.attend(0, torch.from_numpy(q).cuda(), 2, rows, scale=scale).cpu().numpy()
        want, _, size, _ = ref.attend(q, 2, rows, scale)
        near = 4 * 8 * 2.0 ** -24 * size + 2.0 ** -20
        for h in range(2):
            top = np.abs(ref.values("v", 0, h, 400)).max()
            assert np.abs(got[:, 64 * h:64 * h + 64] - want[:, 64 * h:64 * h + 64]).max() <= near * top


def test_attention_weight_on_a_block_of_tiny_values(kt):
    """A softmax that rests on a block whose values are 1e-15 of the others' keeps their relative accuracy."""
    cache, ref, rng = make(kt, 1, 1, 64, 128, 16, [95])
    for i in range(6):
        k = np.full((16, 64), -60.0 if i != 2 else 60.0, np.float32)
        v = (rng.standard_normal((16, 64)) * (1e-15 if i == 2 else 1.0)).astype(np.float32)
        from oracle.kv8_oracle import quantise
        ref.codes["k"][0, 0, 16 * i:16 * i + 16], ref.scales["k"][0, 0, i] = quantise(k)
        ref.codes["v"][0, 0, 16 * i:16 * i + 16], ref.scales["v"][0, 0, i] = quantise(v)
    push(cache, ref)
    q = np.full((1, 64), 1.0, np.float32)  # scores of -480 and 480
    got = cache.attend(0, torch.from_numpy(q).cuda(), 1, 1).cpu().numpy()
    want, _, _, _ = ref.attend(q, 1, 1, 0.125)
    # all scores of the block are equal: what is left is the rounding of a mean of 16 values
    assert np.abs(got - want).max() <= 2.0 ** -20 * np.abs(ref.values("v", 0, 0, 48)[32:]).max()


def test_attention_shows_values_that_are_not_finite(kt):
    """A key or value block of scale NaN makes the rows that see it NaN, and no other head's."""
    cache, ref, rng = make(kt, 1, 2, 64, 256, 16, [200])
    cache.k_scales[0, 0, 0, 3] = float("nan")
    q = torch.randn(1, 8 * 64, device="cuda")
    out = cache.attend(0, q, 8)
    assert bool(out[:, :256].isnan().all()) and bool(out[:, 256:].isfinite().all())
    bad = torch.randn(1, 8 * 64, device="cuda")
    bad[0, 300] = float("inf")  # a query of head 4
    out = cache.attend(0, bad, 8)
    assert bool(out[:, 256:320].isnan().all()) and bool(out[:, 320:].isfinite().all())


@pytest.mark.parametrize("rows", [12, 60])
def test_attention_of_rows_before_a_value_that_is_not_finite(kt, rows):
    """A token of NaN poisons its block of 16 slots: rows before the block stay finite, rows from the
    token on are NaN."""
    from kotensor_b200.kv8 import KVCache8
    for name in "kv":
        cache = KVCache8(1, 1, 2, 64, 128, 16)
        x = {n: torch.randn(rows, 128, device="cuda") for n in "kv"}
        x[name][10, :64] = float("nan")   # slot 36 + 10 = 46 of head 0: the block 32..47
        cache.store(0, torch.randn(36, 128, device="cuda"), torch.randn(36, 128, device="cuda"), 36)
        cache.advance(36)
        cache.store(0, x["k"], x["v"], rows)
        cache.lengths.fill_(28)           # row t sees slots 0..28 + t
        out = cache.attend(0, torch.randn(rows, 512, device="cuda"), 8, rows)
        assert bool(out[:4].isfinite().all()), name
        assert bool(out[4:, :256].isnan().all()) and bool(out[:, 256:].isfinite().all()), name


def test_attention_is_the_same_on_every_run_and_in_a_graph(kt):
    """Equal bits from run to run, on another stream, and when a captured step replays at other lengths."""
    cache, ref, rng = make(kt, 3, 4, 128, 1024, 64, [5, 700, 300])
    q = torch.randn(3, 16 * 128, device="cuda")
    out = cache.attend(0, q, 16, accumulate=True)
    w = cache.weights.clone()
    push(cache, ref)
    assert torch.equal(cache.attend(0, q, 16, accumulate=True), out) and torch.equal(w.nan_to_num(), cache.weights.nan_to_num())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(cache.attend(0, q, 16), out)
    torch.cuda.current_stream().wait_stream(s)
    held = torch.zeros_like(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(0, q, 16, out=held)
    for lengths in ([0, 1, 2], [5, 700, 300], [4, 64, 63]):
        cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        g.replay()
        assert torch.equal(held, cache.attend(0, q, 16)) and bool(held.isfinite().all())


def test_attention_past_32_bit_offsets(kt):
    """A cache of more than 2^32 code bytes: the last sequence's slots are read, and stored, where they are."""
    from kotensor_b200.kv8 import KVCache8
    b, h, d, cap = 3, 8, 128, 1 << 21
    cache = KVCache8(1, b, h, d, cap, 64)
    n = 700
    small = KVCache8(1, 1, h, d, 1024, 64)
    k, v = torch.randn(n, h * d, device="cuda"), torch.randn(n, h * d, device="cuda")
    small.store(0, k, v, n)
    cache.store(0, k.repeat(b, 1), v.repeat(b, 1), n, counts=torch.tensor([0, 0, n], dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.k_codes[0, 2, :, :n], small.k_codes[0, 0, :, :n])
    # the very end of the last sequence
    cache.v_codes[0, 2, :, cap - 64:] = small.v_codes[0, 0, :, :64]
    cache.v_scales[0, 2, :, -1] = small.v_scales[0, 0, :, 0]
    q = torch.randn(b, 32 * d, device="cuda")
    cache.lengths.copy_(torch.tensor([0, 0, n - 1], dtype=torch.int32))
    small.lengths.fill_(n - 1)
    a, e = cache.attend(0, q, 32)[2], small.attend(0, q[2:].contiguous(), 32)[0]
    assert (a - e).abs().max() <= 1e-5 * e.abs().max()
    cache.lengths.copy_(torch.tensor([0, 0, cap - 1], dtype=torch.int32))
    out = cache.attend(0, torch.zeros(b, 32 * d, device="cuda"), 32)[2].reshape(h, 4, d)  # the mean of all values
    total = ((small.v_codes[0, 0, :, :n].double() * small.v_scales[0, 0, :, :n // 64 + 1].double().repeat_interleave(64, 1)[:, :n, None]).sum(1)
             + (small.v_codes[0, 0, :, :64].double() * small.v_scales[0, 0, :, :1, None].double()).sum(1)) / cap
    assert (out.double() - total[:, None]).abs().max() <= 1e-5 * total.abs().max()


@pytest.mark.parametrize("b,h,d,block,lengths,keep,recent", [
    (1, 1, 16, 16, [2], 1, 0),
    (1, 2, 64, 64, [1001], 512, 128),
    (3, 2, 80, 16, [40, 41, 200], 40, 40),        # only the recent ones; one sequence short enough already
    (2, 3, 128, 32, [300, 2000], 299, 0),
    (1, 1, 48, 16, [5000], 3001, 17),
    (2, 8, 128, 64, [1500, 1025], 1024, 100),
    (4, 1, 96, 64, [9, 10, 11, 3000], 10, 3),
])
def test_evict_keeps_what_weighs_most(kt, b, h, d, block, lengths, keep, recent):
    cache, ref, rng = make(kt, b, h, d, max(lengths) + 5, block, lengths, seed=keep)
    w = np.exp(2 * rng.standard_normal(ref.weights.shape)).astype(np.float32)
    w[rng.random(w.shape) < 0.4] = 0.0
    w[rng.random(w.shape) < 0.1] = 1.5            # ties at zero and in the middle
    w[rng.random(w.shape) < 0.05] = -0.0
    for i, n in enumerate(lengths):
        ref.weights[i, :, :n] = w[i, :, :n]
    push(cache, ref)
    before = cache.lengths.clone()
    ref.evict(keep, recent)
    cache.evict_layer(0, keep, recent)
    assert_same(cache, ref)
    assert torch.equal(before, cache.lengths)
    cache.advance(0, limit=keep)
    assert cache.lengths.tolist() == [min(n, keep) for n in lengths]


def test_evict_with_weights_that_are_not_ordinary(kt):
    cache, ref, rng = make(kt, 1, 3, 32, 512, 16, [400])
    w = rng.standard_normal((3, 400)).astype(np.float32)  # negative ones too
    w[0, 50], w[0, 7], w[1, 300], w[2, 9] = np.nan, np.inf, -np.inf, np.nan
    w[2, 20:60] = np.nan
    ref.weights[0, :, :400] = w
    push(cache, ref)
    ref.evict(100, 10)
    cache.evict_layer(0, 100, 10)
    assert_same(cache, ref)


def test_evict_all_equal_weights_keeps_the_lowest_slots(kt):
    cache, ref, rng = make(kt, 1, 2, 64, 4096, 64, [4000])
    ref.weights[:] = 0.25
    push(cache, ref)
    ref.evict(1000, 1)
    cache.evict_layer(0, 1000, 1)
    assert ref.kept(0, 0, 1000, 1)[:999].tolist() != [] and np.array_equal(
        cache.weights[0].cpu().numpy(), ref.weights)
    assert_same(cache, ref)


def test_store_after_evict_continues_the_open_block(kt):
    cache, ref, rng = make(kt, 2, 2, 64, 512, 32, [400, 90])
    for i, n in enumerate([400, 90]):
        ref.weights[i, :, :n] = rng.random((2, n)).astype(np.float32)
    push(cache, ref)
    ref.evict(77, 20)
    ref.lengths[:] = np.minimum(ref.lengths, 77)
    cache.evict(77, 20)
    for _ in range(3):
        k, v = (rng.standard_normal((2, 128), dtype=np.float32) for _ in range(2))
        ref.store(k, v, 1)
        ref.lengths += 1
        cache.store(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        cache.advance()
    assert_same(cache, ref)


def test_layers_are_apart(kt):
    cache, ref, rng = make(kt, 1, 2, 64, 128, 16, [20], layers=3)
    before = [cache.k_codes[l].clone() for l in (0, 2)]
    k = torch.randn(1, 128, device="cuda")
    cache.store(1, k, k)
    assert torch.equal(cache.k_codes[0], before[0]) and torch.equal(cache.k_codes[2], before[1])
    assert bool((cache.k_codes[1, 0, :, 20] != 0).any())


def test_refusals(kt):
    import ctypes
    from kotensor_b200 import _lib
    from kotensor_b200.kv8 import KVCache8
    for bad in (dict(head_dim=24), dict(head_dim=144), dict(head_dim=0), dict(block=48), dict(block=128), dict(batch=0),
                dict(batch=40000), dict(capacity=0), dict(layers=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            KVCache8(**{**dict(layers=1, batch=1, kv_heads=1, head_dim=64, capacity=64), **bad})
    cache = KVCache8(2, 2, 2, 64, 100, 32)
    assert cache.capacity == 128
    x = torch.zeros(2, 128, device="cuda")
    with pytest.raises(ValueError):
        cache.store(2, x, x)
    with pytest.raises(ValueError):
        cache.store(0, x[:1], x)
    with pytest.raises(ValueError):
        cache.store(0, x.double(), x)
    with pytest.raises(ValueError):
        cache.store(0, x.cpu(), x)
    with pytest.raises(ValueError):
        cache.store(0, x, x, counts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        cache.store(0, x.t().contiguous().t(), x)
    with pytest.raises(ValueError):
        cache.attend(0, x, 3)
    with pytest.raises(ValueError):
        cache.attend(0, torch.zeros(2, 192, device="cuda"), 3)   # 3 heads over 2
    with pytest.raises(ValueError):
        cache.attend(0, x, 2, accumulate=True)                    # no weights kept
    with pytest.raises(ValueError):
        cache.attend(0, x, 2, out=torch.zeros(2, 64, device="cuda"))
    with pytest.raises(ValueError):
        cache.evict_layer(0, 10, 2)
    tracked = KVCache8(1, 2, 2, 64, 100, 32, track_weights=True)
    for keep, recent in ((0, 0), (5, 6), (5, -1)):
        with pytest.raises(ValueError):
            tracked.evict_layer(0, keep, recent)
    lib, h = _lib.load(), kt.Context.get().handle
    s = _lib.KtKv8Cache.from_buffer_copy(cache._layer[0][0])
    for field, value in (("k_codes", 0), ("lengths", 0), ("head_dim", 40), ("block", 8), ("capacity", 33), ("batch", 0),
                         ("kv_heads", 0)):
        t = _lib.KtKv8Cache.from_buffer_copy(s)
        setattr(t, field, value)
        assert lib.kt_kv8_store(h, ctypes.byref(t), x.data_ptr(), x.data_ptr(), 128, 128, 1, None, None, None) == 1
    assert lib.kt_kv8_store(h, ctypes.byref(s), x.data_ptr(), x.data_ptr(), 100, 128, 1, None, None, None) == 1
    assert lib.kt_kv8_store(h, ctypes.byref(s), None, None, 128, 128, 1, None, None, None) == 1
    assert lib.kt_kv8_store(h, ctypes.byref(s), None, None, 128, 128, 0, None, None, None) == 0
    assert lib.kt_kv8_store(h, ctypes.byref(s), x.data_ptr(), x.data_ptr(), 128, 128, -1, None, None, None) == 1
    assert lib.kt_kv8_attention(h, ctypes.byref(s), x.data_ptr(), 128, x.data_ptr(), 1, None, 2, 1.0, 0, None, None) == 1
    assert lib.kt_kv8_scratch_bytes(0, 1, 1, 1, 64, 64, 0) == 0
