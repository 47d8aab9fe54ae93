"""Calls of the paged cache at its edges, against the definitions in 64 bits (oracle/paged_oracle.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_gpu import BF16, FP16, LLAMA, MQA, ODD, QWEN, WIDE, check_attend, filled, no_wait_ran_out, put, queries, trees  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout,rows,lengths", [(LLAMA, 1, [3000, 5]), (LLAMA, 1, [300]), (QWEN, 9, [700, 64]), (LLAMA, 70, [900, 0]), (MQA, 40, [2000])])
def test_results_in_the_queries_place(kt, layout, rows, lengths):
    cache = filled(layout, 32, BF16, lengths, rows)
    put(cache, rows)
    q = queries(cache, layout[0], rows)
    want = cache.attend(0, q, layout[0], rows)
    for _ in range(3):
        mine = q.clone()
        assert cache.attend(0, mine, layout[0], rows, out=mine) is mine
        assert torch.equal(mine, want)
    if len(q) == 1:  # (one row has no gaps, whatever its stride)
        part = torch.empty(1, q.shape[1] + 64, dtype=BF16, device="cuda")[:, :q.shape[1]]
        part.copy_(q)
        assert torch.equal(cache.attend(0, part, layout[0], rows, out=part), want)
    room = torch.zeros(q.numel() + 8, dtype=BF16, device="cuda")
    beside = room[8:].view(q.shape)
    beside.copy_(q)
    with pytest.raises(ValueError, match="overlap"):
        cache.attend(0, beside, layout[0], rows, out=room[:-8].view(q.shape))
    assert torch.equal(beside, q)


def poke(cache, which, slot, dim, value, b=0):
    """One value of every head in a slot."""
    page = int(cache.table[b, slot // cache.page])
    getattr(cache, which)[0, page, :, slot % cache.page, dim] = value


@pytest.mark.parametrize("layout,dtype,rows,held", [
    (LLAMA, BF16, 1, 700), (QWEN, FP16, 1, 301), (QWEN, BF16, 3, 5000), (ODD, FP16, 2, 400), (LLAMA, BF16, 70, 700), (QWEN, FP16, 30, 700),
    (QWEN, BF16, 300, 130), (MQA, FP16, 16, 900), (MQA, BF16, 130, 5000), (ODD, BF16, 100, 400), (WIDE, FP16, 24, 600),
])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_value_that_is_not_finite_reaches_its_dim_alone(kt, layout, dtype, rows, held, bad):
    """Wherever its slot lies in a tile and however the work is cut: NaN in the value's dim for the rows that see it,
    and every other bit as with a 0 in its place."""
    heads, kv, d = layout
    cache = filled(layout, 32, dtype, [held, held // 2], rows, poison=True)
    put(cache, rows)
    q = queries(cache, heads, rows)
    new = min(rows - 1, 5)
    for slot, dim in ((3, 5), (held // 2, d - 1), (held - 1, 0), (held + new, 33)):
        poke(cache, "values", slot, dim, 0.0)
        want = cache.attend(0, q, heads, rows).view(2, rows, heads, d).clone()
        assert torch.isfinite(want).all()
        sees = torch.arange(rows, device="cuda") >= slot - held
        want[0, sees, :, dim] = float("nan")
        poke(cache, "values", slot, dim, bad)
        for out in (None, torch.empty(2 * rows, heads * d, device="cuda")):
            got = cache.attend(0, q, heads, rows, out=out).view(want.shape).to(dtype)
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
        poke(cache, "values", slot, dim, 0.25)


@pytest.mark.parametrize("layout,dtype,rows", [(LLAMA, BF16, 1), (QWEN, FP16, 2), (MQA, BF16, 16), (MQA, FP16, 40), (LLAMA, BF16, 65)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_value_of_no_weight_that_is_not_finite(kt, layout, dtype, rows, bad):
    """Scores of the first 400 slots lie so far below the others that their powers are 0; what is there is seen all the same."""
    heads, kv, d = layout
    cache = filled(layout, 64, dtype, [1200], rows)
    put(cache, rows)
    q = torch.ones(rows, heads * d, dtype=dtype, device="cuda")
    slot = torch.arange(400)
    cache.keys[0, cache.table[0].cpu()[slot // 64].long(), :, slot % 64] = -60.0
    for at in (7, 390):
        poke(cache, "values", at, 9, bad)
        got = cache.attend(0, q, heads, rows).view(rows, heads, d)
        poke(cache, "values", at, 9, 0.0)
        want = cache.attend(0, q, heads, rows).view(rows, heads, d)
        assert torch.isnan(got[..., 9]).all() and torch.equal(got[..., :9], want[..., :9]) and torch.equal(got[..., 10:], want[..., 10:])


@pytest.mark.parametrize("layout,dtype,rows", [(LLAMA, BF16, 5), (QWEN, FP16, 60)])
def test_a_key_that_is_not_a_number_reaches_all_dims_of_its_head(kt, layout, dtype, rows):
    heads, kv, d = layout
    cache = filled(layout, 64, dtype, [300], rows)
    put(cache, rows)
    q = queries(cache, heads, rows)
    want = cache.attend(0, q, heads, rows).view(rows, kv, heads // kv, d)
    for slot in (10, 299, 302):
        page = int(cache.table[0, slot // 64])
        was = cache.keys[0, page, 1, slot % 64, 3].clone()
        cache.keys[0, page, 1, slot % 64, 3] = float("nan")
        got = cache.attend(0, q, heads, rows).view(want.shape)
        sees = torch.arange(rows, device="cuda") >= slot - 300
        assert torch.isnan(got[sees][:, 1]).all() and torch.equal(got[~sees], want[~sees])
        assert torch.equal(got[:, [h for h in range(kv) if h != 1]], want[:, [h for h in range(kv) if h != 1]])
        cache.keys[0, page, 1, slot % 64, 3] = was


@pytest.mark.parametrize("rows", [6, 70])
def test_drafted_values_that_are_not_finite(kt, rows):
    """Some of a tree's nodes see them and some do not, in several dims and slots of a tile."""
    from kotensor_b200.paged import draft_tree
    heads, kv, d = LLAMA
    _, visible = draft_tree(trees(1, rows, seed=5))
    seen = torch.from_numpy(visible).cuda()
    cache = filled(LLAMA, 64, BF16, [100], rows, poison=True)
    put(cache, rows)
    spots = [(1, 5, float("inf")), (1, 70, float("nan")), (3, 6, -float("inf")), (4, 127, float("nan")), (rows - 1, 0, float("inf"))]
    for u, dim, _ in spots:
        poke(cache, "values", 100 + u, dim, 0.0)
    q = queries(cache, heads, rows)
    want = cache.attend(0, q, heads, rows, visible=seen).view(rows, heads, d).clone()
    for u, dim, bad in spots:
        poke(cache, "values", 100 + u, dim, bad)
        sees = (seen[0, :, u // 32] >> (u % 32) & 1).bool()
        want[sees, :, dim] = float("nan")
    got = cache.attend(0, q, heads, rows, visible=seen).view(want.shape)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("rows", [1, 5, 60])
def test_queries_of_rows_past_the_last_slot_are_zeros(kt, rows):
    heads, kv, d = QWEN
    cache = filled(QWEN, 16, BF16, [46, 5, 48], 0)
    assert cache.capacity == 48
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(3 * rows, n * d, generator=gen).cuda() for n in (heads, kv, kv))
    out = torch.full((3 * rows, heads * d), float("nan"), dtype=BF16, device="cuda")
    cache.append(0, q, k, v, torch.ones(d // 2, device="cuda"), rows, out=out)
    lines = out.view(3, rows, -1)
    for b, room in enumerate((2, 43, 0)):
        assert (lines[b, :room].abs().sum(-1) > 0).all() and not lines[b, room:].any()
    assert int(cache.status) != 0


def test_a_batch_that_the_pool_cannot_hold_takes_no_pages(kt, oracle):
    from test_decoder_paged_gpu import decoder
    prompts = np.random.default_rng(3).integers(0, 700, (2, 50)).tolist()
    d = decoder("int4_gqa", max_seq=128, batch=2, kv_bits=16, kv_page=16, kv_pages=7)
    with pytest.raises(ValueError, match="8 pages wanted, 7 are free"):
        d.prefill(prompts)
    with pytest.raises(ValueError, match="pages wanted"):
        d.generate_batch(prompts, 20)
    assert d.cache.free_pages == 7 and d.length == 0
    got = d.prefill([p[:40] for p in prompts])  # three pages each
    assert d.cache.free_pages == 1 and torch.equal(got, decoder("int4_gqa", max_seq=128, batch=2, kv_bits=16, kv_page=16).prefill(
        [p[:40] for p in prompts]))


def test_a_drafted_text_that_lost_tokens_leaves_the_prompt(kt, oracle):
    from test_decoder_paged_gpu import decoder
    prompts = np.random.default_rng(13).integers(0, 700, (2, 12)).tolist()
    d, e = (decoder("int4_gqa", max_seq=96, batch=2, kv_bits=16) for _ in range(2))
    d.cache.status.fill_(1)  # as a token without a page would
    with pytest.raises(ValueError, match="dropped"):
        d.generate_drafted(prompts, 30)
    e.prefill(prompts)
    assert d.length == 12 == int(d.position) and d.cache.lengths.tolist() == [12, 12]
    assert torch.equal(d.step([5, 6]), e.step([5, 6])) and d.cache.lengths.tolist() == [13, 13]


def test_many_items_of_one_tile(kt):
    """Items of 72 vectors over one tile, several to a CTA: the second stream has no tile in any of them."""
    heads, rows = MQA[0], 9
    cache = filled(MQA, 32, BF16, [(37 * i) % 119 for i in range(450)], rows, poison=True)
    counts = torch.tensor([rows - i % 3 for i in range(450)], dtype=torch.int32).cuda()
    put(cache, rows, counts)
    q = queries(cache, heads, rows)
    got = cache.attend(0, q, heads, rows, counts)
    assert all(torch.equal(cache.attend(0, q, heads, rows, counts), got) for _ in range(20))
    check_attend(cache, q, heads, rows, got, counts)


@pytest.mark.parametrize("layout,rows,held", [((8, 2, 64), 10, 1300), ((8, 1, 128), 12, 1200), ((14, 2, 64), 40, 900), ((8, 2, 128), 48, 1000),
                                              (MQA, 1, 2000), (QWEN, 6, 1100)])
@pytest.mark.parametrize("dtype,rising", [(BF16, True), (FP16, True), (FP16, False)])
def test_largest_scores_late_in_a_text(kt, layout, rows, held, dtype, rising):
    """Scores that rise by more than 2^8 every few hundred slots, for some rows and not for others (with rows of both
    signs some fall): references move in the middle of a run, in some vectors of a warp, in one stream or both."""
    heads, kv, d = layout
    batch = 60 if rows == 10 else 9 if rows == 12 else 2  # enough of the small ones for the kernel of many vectors
    cache = filled(layout, 32, dtype, [held - 7 * b for b in range(batch)], rows, poison=True)
    for b in range(batch):
        slot = torch.arange(held - 7 * b)
        level = (slot // 200 if rising else (held - slot) // 150).float() - 3.0
        page = cache.table[b].cpu()[slot // 32].long()
        noise = cache.keys[0, page, :, slot % 32].float() * 0.1
        cache.keys[0, page, :, slot % 32] = (level.cuda()[:, None, None] + noise).to(dtype)
    put(cache, rows)
    gen = torch.Generator().manual_seed(9)
    slope = torch.tensor([1.0, -0.5, 0.0, 2.0, 1.5])[torch.randint(0, 5, (batch * rows, heads, 1), generator=gen)]
    q = (slope + 0.1 * torch.randn(batch * rows, heads, d, generator=gen)).reshape(batch * rows, -1).to(dtype).cuda()
    for scale in (None, -0.1):
        got = cache.attend(0, q, heads, rows, scale=scale, out=torch.empty(q.shape, device="cuda"))
        assert torch.equal(got, cache.attend(0, q, heads, rows, scale=scale, out=torch.empty_like(got)))
        some = cache.sequences(0, 2)  # (the oracle's time)
        check_attend(some, q[:2 * rows], heads, rows, got[:2 * rows], scale=scale)


@pytest.mark.parametrize("layout,rows", [(QWEN, 1), (LLAMA, 5), (LLAMA, 40), (MQA, 20)])
def test_a_scale_of_zero_weighs_all_alike(kt, layout, rows):
    heads, kv, d = layout
    cache = filled(layout, 32, FP16, [90, 300], rows, poison=True)
    put(cache, rows)
    q = queries(cache, heads, rows)
    for scale in (0.0, -0.0, 1e-44):
        check_attend(cache, q, heads, rows, cache.attend(0, q, heads, rows, scale=scale), scale=scale)


@pytest.mark.parametrize("name,batch", [("int4_gqa", 2), ("int8_tied_mha", 1)])
def test_true_drafts_are_accepted(kt, oracle, name, batch):
    """A text told in full is accepted seven drafts at a time behind a wrong branch; a text told wrong takes one pass a
    token.  Both say the same.  Of 47 tokens after the first, five passes give 8 each; the sixth may have 7 nodes, one of
    which the wrong branch takes, and gives 6; the seventh gives the last."""
    from test_decoder_paged_gpu import decoder
    prompts = np.random.default_rng(14).integers(0, 700, (batch, 12)).tolist()
    options = dict(max_seq=160, batch=batch, kv_bits=16, kv_page=16)
    wrong = decoder(name, **options)
    truth = wrong.generate_drafted(prompts, 48, nodes=12, draft=lambda text: [[700, 701, 702], [703]])
    assert wrong.passes == 47 and not any(t in (700, 703) for text in truth for t in text)

    def told(text):
        for p, t in zip(prompts, truth):
            if text[:12] == p and text[12:] == t[:len(text) - 12]:
                after = t[len(text) - 12:][:7]
                return [after[:2] + [700], after]
        raise AssertionError("another text")

    d = decoder(name, **options)
    assert d.generate_drafted(prompts, 48, nodes=12, draft=told) == truth
    assert d.passes == 7
