"""Calls of the 8-bit key/value cache one after another: lengths that follow the
counts of a store, scratch over prompts of many lengths, a cache used first inside
a captured graph, and views of some sequences."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def test_advance_takes_counts_as_the_store_does(kt):
    """Counts above the rows and below zero: lengths move by the tokens that were stored, over several calls, so
    what is attended to is what the oracle holds (tolerance of the attention: test_kv8_gpu.py)."""
    from test_kv8_gpu import assert_same, make
    b, h, d, heads, rows = 4, 2, 64, 8, 7
    cache, ref, rng = make(kt, b, h, d, 128, 16, [0, 10, 33, 60])
    for counts in ([40, -2, 3, 0], [7, 8, -100, 2 ** 31 - 1], [-2 ** 31, 5, 7, 6]):
        k, v = (rng.standard_normal((b * rows, h * d), dtype=np.float32) for _ in range(2))
        dev = torch.tensor(counts, dtype=torch.int32, device="cuda")
        cache.store(0, cuda(k), cuda(v), rows, counts=dev)
        assert not ref.store(k, v, rows, counts)
        q = rng.standard_normal((b * rows, heads * d), dtype=np.float32)
        got = cache.attend(0, cuda(q), heads, rows, counts=dev).cpu().numpy()
        want, _, size, top = ref.attend(q, heads, rows, d ** -0.5, counts)
        assert np.abs(got - want).max() <= (4 * d ** 0.5 * 2.0 ** -24 * size + 2.0 ** -20) * top
        cache.advance(rows, counts=dev)
        ref.lengths += np.clip(counts, 0, rows).astype(np.int32)
        assert cache.lengths.tolist() == ref.lengths.tolist()
        assert_same(cache, ref)


def test_advance_stays_between_zero_and_its_limit(kt):
    from kotensor_b200.kv8 import KVCache8
    cache = KVCache8(1, 4, 1, 16, 64, 16)
    cache.lengths.copy_(torch.tensor([0, 5, 60, 64], dtype=torch.int32))
    cache.advance(10)
    assert cache.lengths.tolist() == [10, 15, 64, 64]
    cache.advance(counts=torch.tensor([3, 70, -4, 1], dtype=torch.int32, device="cuda"))  # rows not given: as counted
    assert cache.lengths.tolist() == [13, 64, 64, 64]
    cache.advance(0, counts=torch.tensor([3, 3, 3, 3], dtype=torch.int32, device="cuda"))
    assert cache.lengths.tolist() == [13, 64, 64, 64]
    cache.advance(0, limit=20)
    assert cache.lengths.tolist() == [13, 20, 20, 20]
    cache.advance(2 ** 31 - 1)
    assert cache.lengths.tolist() == [64] * 4
    cache.lengths.fill_(5)
    cache.advance(-9)
    assert cache.lengths.tolist() == [0] * 4
    with pytest.raises(ValueError):
        cache.advance(-1, counts=torch.ones(4, dtype=torch.int32, device="cuda"))


def test_scratch_does_not_pile_up_over_prompt_lengths(kt):
    """Attention with weights over prompts of ever more rows: what the cache holds is bounded by the scratch of the
    longest call and of a single-token step, whatever came before (in bytes asked for: the allocator's blocks may
    be larger than what is asked of them)."""
    import gc
    from kotensor_b200 import _lib
    from kotensor_b200.kv8 import KVCache8
    b, h, d, heads, cap = 2, 8, 128, 32, 4096
    cache = KVCache8(1, b, h, d, cap, 64, track_weights=True)
    q = torch.randn(b * 3000, heads * d, device="cuda")
    out = torch.empty_like(q)
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    lengths = [1] + list(range(200, 3001, 200))
    for rows in lengths:
        cache.attend(0, q[:b * rows], heads, rows, out=out[:b * rows], accumulate=True)
        cache.lengths.zero_()
    gc.collect()
    torch.cuda.synchronize()
    need = [_lib.load().kt_kv8_scratch_bytes(b, rows, heads, h, d, cap, 1) for rows in (1, max(lengths))]
    assert torch.cuda.memory_stats()["requested_bytes.all.current"] - before <= sum(need) + 4096
    # a step captured in a graph keeps its scratch through longer prompts
    step = q[:b].contiguous()
    held = torch.empty_like(step)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(0, step, heads, out=held)
    big = KVCache8(1, b, h, d, cap, 64, track_weights=True)
    cache.attend(0, torch.randn(b * 3500, heads * d, device="cuda"), heads, 3500, accumulate=True)
    cache.lengths.fill_(1234)
    big.lengths.fill_(1234)
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        x = getattr(cache, name)
        x.copy_(torch.randint(-127, 128, x.shape, device="cuda") if x.dtype == torch.int8 else torch.rand(x.shape, device="cuda"))
        getattr(big, name).copy_(x)
    g.replay()
    assert torch.equal(held, big.attend(0, step, heads))


def test_a_graph_that_is_the_first_to_call_leaves_the_scratch_usable(kt):
    """The first call of a cache is captured, in a pool whose free memory is full of ones; a call outside the graph
    comes before the first replay."""
    from kotensor_b200.kv8 import KVCache8
    pool = torch.cuda.graph_pool_handle()
    dirt = torch.cuda.CUDAGraph()
    with torch.cuda.graph(dirt, pool=pool):
        x = torch.full((64 << 20,), -1, dtype=torch.int8, device="cuda")
    dirt.replay()
    torch.cuda.synchronize()
    del x
    one, two = (KVCache8(1, 1, 2, 64, 8192, 16) for _ in range(2))
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        x = getattr(one, name)
        x.copy_(torch.randint(-127, 128, x.shape, device="cuda") if x.dtype == torch.int8 else torch.rand(x.shape, device="cuda"))
        getattr(two, name).copy_(x)
    for c in (one, two):
        c.lengths.fill_(8000)
    q = torch.randn(1, 512, device="cuda")
    held = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool):
        one.attend(0, q, 8, out=held)
    want = two.attend(0, q, 8)
    assert torch.equal(one.attend(0, q, 8, out=torch.zeros_like(q)), want)
    g.replay()
    assert torch.equal(held, want)
    assert torch.equal(one.attend(0, q, 8), want)


def test_a_view_of_some_sequences(kt):
    """`sequences` stores, attends, advances and evicts on its part of the buffers alone."""
    from test_kv8_gpu import assert_same, make, push
    cache, ref, rng = make(kt, 4, 2, 64, 256, 32, [3, 70, 33, 100])
    part, part_ref, _ = make(kt, 2, 2, 64, 256, 32, [70, 33])
    for name in ("codes", "scales", "tail"):
        for n in "kv":
            getattr(part_ref, name)[n][:] = getattr(ref, name)[n][1:3]
    part_ref.weights[:] = np.abs(rng.standard_normal(part_ref.weights.shape)).astype(np.float32)
    ref.weights[1:3] = part_ref.weights
    push(cache, ref)
    push(part, part_ref)
    view = cache.sequences(1, 3)
    k = cuda(rng.standard_normal((2 * 5, 128), dtype=np.float32))
    q = cuda(rng.standard_normal((2 * 5, 512), dtype=np.float32))
    results = []
    for c in (view, part):
        c.store(0, k, k, 5)
        results.append(c.attend(0, q, 8, 5, accumulate=True))
        c.advance(5)
        c.evict(40, 8)
    assert torch.equal(*results)
    assert cache.lengths.tolist() == [3, 40, 38, 100] and part.lengths.tolist() == [40, 38]
    for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail", "weights"):
        a, b = getattr(cache, name)[0], getattr(part, name)[0]
        assert torch.equal(a[1:3].nan_to_num(), b.nan_to_num())
    for n in "kv":  # the others are as they were
        for name in ("codes", "scales", "tail"):
            got = getattr(cache, f"{n}_{name}")[0].cpu().numpy()[[0, 3]]
            assert np.array_equal(got, getattr(ref, name)[n][[0, 3]], equal_nan=name != "codes")
