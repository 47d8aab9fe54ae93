"""PagedKVCache on the GPU against its definitions in 64 bits (oracle/paged_oracle.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
# heads, kv_heads, head_dim
LLAMA, QWEN, MHA, MQA, WIDE = (32, 8, 128), (14, 2, 64), (12, 12, 64), (8, 1, 128), (24, 2, 96)
ODD = (15, 5, 80)


@pytest.fixture(autouse=True)
def no_wait_ran_out(kt):
    yield
    torch.cuda.synchronize()
    assert kt.Context.get(0).take_error() == 0


def filled(layout, page, dtype, lengths, room, layers=1, seed=0, spare=2, poison=False):
    """A cache whose sequences hold `lengths` tokens, with pages for `room` more in a shuffled
    table.  poison: every slot that holds no token is NaN."""
    from kotensor_b200.paged import PagedKVCache
    _, kv, d = layout
    gen = torch.Generator().manual_seed(seed)
    batch = len(lengths)
    width = max(1, -(-(max(lengths) + room) // page))
    pool = batch * width + spare
    cache = PagedKVCache(layers, batch, kv, d, pool, width * page, page, dtype)
    cache.table.copy_(torch.randperm(pool, generator=gen)[:batch * width].reshape(batch, width).int())
    for x in (cache.keys, cache.values):
        x.copy_(torch.randn(x.shape, generator=gen).to(dtype))
        if poison:
            used = torch.zeros(pool, page, dtype=torch.bool)
            for b, n in enumerate(lengths):
                s = torch.arange(n)
                used[cache.table[b].cpu()[s // page].long(), s % page] = True
            x.masked_fill_(~used[None, :, None, :, None].cuda(), float("nan"))
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    return cache


def trees(batch, rows, seed=0):
    """Parents of random drafted trees: chains and branches."""
    rng = np.random.default_rng(seed)
    p = np.array([[-1] + [int(rng.integers(max(0, t - 1 - t // 2), t)) for t in range(1, rows)] for _ in range(batch)])
    return p


def put(cache, rows, counts=None, seed=1, layer=0):
    """Appends random new tokens without queries, unrotated."""
    gen = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(cache.batch * rows, cache.kv_heads * cache.head_dim, generator=gen).cuda() for _ in range(2))
    cache.append(layer, None, k, v, torch.zeros(cache.head_dim // 2, device="cuda"), rows, counts)


def check_attend(cache, q, heads, rows, got, counts=None, visible=None, layer=0, scale=None):
    from oracle import paged_oracle as PO
    cpu = lambda x: None if x is None else x.cpu()  # noqa: E731
    want, size, spread = PO.attend(cache.keys[layer].cpu(), cache.values[layer].cpu(), cache.table.cpu(), cache.lengths.cpu(),
                                   q.cpu(), heads, rows, cpu(counts), cpu(visible), scale)
    # A probability is rounded to the cache's type: half a step of it, of the sum of |p v|.  A score is a sum of
    # head_dim products that the tensor cores may truncate at every one: head_dim 2^-23 of the sum of |q k| (`spread`),
    # twice, since the score's error is also the denominator's.  The fp32 sums over the slots are truncated at
    # every 16 of them; exp2 and the rest: 2^-20.  Then the result's own rounding.
    half = torch.finfo(cache.dtype).eps / 2
    n = int(cache.lengths.max()) + rows
    bound = size * (half * 1.01 + 2 * cache.head_dim * 2.0 ** -23 * spread + n * 2.0 ** -26 + 2.0 ** -20) + 2.0 ** -24
    if got.dtype != torch.float32:
        bound = bound * (1 + half) + half * want.abs()
    error = (got.cpu().double().reshape(want.shape) - want).abs()
    assert torch.isfinite(got).all()
    assert (error <= bound).all(), float((error / bound).max())


def queries(cache, heads, rows, seed=2, sharp=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (sharp * torch.randn(cache.batch * rows, heads * cache.head_dim, generator=gen)).to(cache.dtype).cuda()


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("layout,page,dtype,lengths,rows,far", [
    (LLAMA, 64, BF16, [0, 63, 64], 1, 0), (QWEN, 16, FP16, [5], 40, 0), (MHA, 32, BF16, [31, 0], 33, 1000003),
    (MQA, 128, FP16, [127, 128, 300], 7, 0), (WIDE, 16, BF16, [15], 1, 7654321), (ODD, 64, FP16, [1, 60], 130, 90000),
])
@pytest.mark.parametrize("strided", [False, True])
def test_append_rotates_and_stores(kt, layout, page, dtype, lengths, rows, far, strided):
    from oracle import paged_oracle as PO
    heads, kv, d = layout
    cache = filled(layout, page, dtype, lengths, rows, layers=2)
    before = [x.clone() for x in (cache.keys, cache.values)]
    gen = torch.Generator().manual_seed(3)
    n = len(lengths) * rows
    fused = torch.randn(n, (heads + 2 * kv) * d + (3 if strided else 0), generator=gen).cuda()
    fused = fused[:, 1:-2] if strided else fused  # rows that start off a 16-byte boundary
    q, k, v = fused.split([heads * d, kv * d, kv * d], 1)
    inv_freq = (10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().cuda()
    depths = None
    if far:
        depths = torch.randint(0, far, (len(lengths), rows), generator=gen).int().cuda()
    counts = torch.tensor([max(0, rows - 2 * i) for i in range(len(lengths))], dtype=torch.int32).cuda() if rows > 1 else None
    out = cache.append(1, q, k, v, inv_freq, rows, counts, depths)
    half, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25
    assert torch.equal(cache.keys[0], before[0][0]) and torch.equal(cache.values[0], before[1][0])
    touched = torch.zeros(cache.keys.shape[1:4:2], dtype=torch.bool)
    for b, held in enumerate(lengths):
        m = rows if counts is None else int(counts[b])
        line = slice(b * rows, b * rows + m)
        at = held + (torch.arange(m) if depths is None else depths[b, :m].cpu())
        where = PO.slots(cache.table.cpu(), b, held + m, page, cache.pages)[held:]
        pages, places = (torch.tensor([w[i] for w in where], dtype=torch.long) for i in (0, 1))
        touched[pages, places] = True
        for x, h, got in ((q, heads, out[line].cpu()), (k, kv, cache.keys[1].cpu()[pages, :, places])):
            x = x[line].cpu().reshape(m, h, d)
            want = PO.rotate(x, at, inv_freq.cpu())
            # angle, sine and cosine, products and sum in fp32: each at most 2^-23 of the pair's |x| + |y|
            pair = x.double().abs().reshape(m, h, 2, -1).sum(2).repeat(1, 1, 2)
            bound = pair * 2.0 ** -21 + half * want.abs() * 1.001 + tiny
            assert ((got.double().reshape(m, h, d) - want).abs() <= bound).all()
        assert torch.equal(cache.values[1].cpu()[pages, :, places], v[line].cpu().reshape(m, kv, d).to(dtype))
        assert not out[b * rows + m:(b + 1) * rows].any()
    for x, was in ((cache.keys, before[0]), (cache.values, before[1])):  # nothing else has changed
        assert torch.equal(x[1].transpose(1, 2)[~touched.cuda()], was[1].transpose(1, 2)[~touched.cuda()])
    assert int(cache.status) == 0


def test_append_without_a_page_drops_the_token(kt):
    cache = filled(QWEN, 16, BF16, [14, 30, 3], 2)  # room for 32 slots each
    cache.table[0, 1] = -1
    cache.table[2, 0] = cache.pages
    before = cache.keys.clone()
    put(cache, 4)
    was = before.transpose(2, 3)[0]
    now = cache.keys.transpose(2, 3)[0]
    changed = [tuple(x) for x in (was != now).any(-1).any(-1).nonzero().tolist()]
    want = [(int(cache.table[0, 0]), 14), (int(cache.table[0, 0]), 15), (int(cache.table[1, 1]), 14), (int(cache.table[1, 1]), 15)]
    assert sorted(changed) == sorted(want)
    assert int(cache.status) != 0
    cache.reset()
    assert int(cache.status) == 0 and not cache.lengths.any()


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("layout,page,lengths,rows", [
    (LLAMA, 64, [0], 1), (LLAMA, 64, [63, 1, 64, 700], 1), (QWEN, 16, [300], 1), (MHA, 32, [5, 0, 130], 1),
    (MQA, 128, [1000, 127], 1), (WIDE, 16, [17, 200], 1), (ODD, 64, [64, 65], 1), (QWEN, 32, [1500, 3, 0, 40, 41], 1),
    (LLAMA, 16, [40, 0], 5), (QWEN, 64, [100], 3), (MHA, 64, [70], 50), (MQA, 32, [33, 250], 17), (WIDE, 128, [3], 45),
    (ODD, 16, [0, 90], 70), (LLAMA, 32, [0], 200), (QWEN, 128, [10, 333], 129),
])
def test_attention_in_order(kt, layout, page, lengths, rows, dtype):
    cache = filled(layout, page, dtype, lengths, rows, poison=True)
    put(cache, rows)
    q = queries(cache, layout[0], rows)
    check_attend(cache, q, layout[0], rows, cache.attend(0, q, layout[0], rows))


@pytest.mark.parametrize("layout,page,dtype", [((6, 2, 112), 16, BF16), ((40, 1, 64), 64, FP16), ((130, 1, 64), 32, BF16),
                                               ((3, 3, 96), 128, FP16), ((9, 3, 80), 16, BF16)])
@pytest.mark.parametrize("rows", [1, 9, 65, 300])
def test_padded_batches_in_order(kt, layout, page, dtype, rows):
    """Prompts of unlike lengths in one call: rows behind a sequence's own give zeros and are not seen."""
    heads, kv, d = layout
    counts = torch.tensor([rows, 0, max(1, rows // 2), rows + 5, -3], dtype=torch.int32).cuda()
    cache = filled(layout, page, dtype, [7, 40, 0, 129, 64], rows, poison=True)
    put(cache, rows, counts)
    q = queries(cache, heads, rows)
    out = torch.full_like(q, float("nan"))
    cache.attend(0, q, heads, rows, counts, out=out)
    lines = out.view(5, rows, -1)
    assert not lines[1].any() and not lines[2, max(1, rows // 2):].any() and not lines[4].any()
    check_attend(cache, q, heads, rows, out, counts)


def test_rows_past_the_last_slot_are_no_tokens(kt):
    heads, kv, d = QWEN
    for rows in (5, 60):
        cache = filled(QWEN, 16, BF16, [30, 5], 2, poison=True)  # 32 slots each
        assert cache.capacity == 32
        put(cache, rows)
        assert int(cache.status) != 0
        q = queries(cache, heads, rows)
        out = cache.attend(0, q, heads, rows)
        assert not out.view(2, rows, -1)[0, 2:].any() and not out.view(2, rows, -1)[1, 27:].any()
        check_attend(cache, q, heads, rows, out)
        cache.advance(rows)
        assert cache.lengths.tolist() == [32, min(32, 5 + rows)]
        assert not cache.attend(0, q, heads, rows).view(2, rows, -1)[0].any()  # a full sequence has no room for tokens


@pytest.mark.parametrize("layout,page,lengths,rows,dtype", [
    (LLAMA, 64, [100, 0, 513], 33, BF16), (QWEN, 16, [64, 7], 2, FP16), (QWEN, 32, [500], 64, BF16), (MHA, 128, [20, 21], 31, FP16),
    (MQA, 64, [0], 100, BF16), (WIDE, 16, [250, 3], 61, BF16), (ODD, 32, [31, 32, 33], 40, FP16), (LLAMA, 128, [1000], 130, FP16),
])
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_of_drafted_trees(kt, layout, page, lengths, rows, dtype, ragged):
    from kotensor_b200.paged import draft_tree
    cache = filled(layout, page, dtype, lengths, rows, poison=True)
    counts = torch.tensor([max(0, rows - 7 * i - 1) for i in range(len(lengths))], dtype=torch.int32).cuda() if ragged else None
    put(cache, rows, counts)
    _, visible = draft_tree(trees(len(lengths), rows))
    visible = torch.from_numpy(visible).cuda()
    q = queries(cache, layout[0], rows)
    check_attend(cache, q, layout[0], rows, cache.attend(0, q, layout[0], rows, counts, visible), counts, visible)


@pytest.mark.parametrize("tokens", [130, 250, 390, 513, 640])
@pytest.mark.parametrize("batch,rows", [(3, 7), (20, 9), (41, 18)])
def test_attention_however_the_work_is_cut(kt, tokens, batch, rows):
    """Items of one to six tiles, alone in a CTA, several to one or shared by some."""
    cache = filled((8, 2, 64), 32, BF16, [max(0, tokens - 97 * (i % 4)) for i in range(batch)], rows, poison=True)
    put(cache, rows)
    q = queries(cache, 8, rows)
    check_attend(cache, q, 8, rows, cache.attend(0, q, 8, rows))


@pytest.mark.parametrize("layout,rows,dtype", [(MQA, 1, BF16), (MQA, 33, BF16), (QWEN, 1, FP16), (QWEN, 45, FP16), (LLAMA, 3, BF16)])
def test_a_long_context(kt, layout, rows, dtype):
    """50021 tokens against 64 bits on the GPU; the tolerance of check_attend."""
    heads, kv, d = layout
    held, n = 50021, 50021 + rows
    cache = filled(layout, 64, dtype, [held], rows)
    put(cache, rows)
    q = queries(cache, heads, rows)
    got = cache.attend(0, q, heads, rows).reshape(rows, kv, -1, d).double()
    slot = torch.arange(n, device="cuda")
    page = cache.table[0, slot // 64].long()
    half = torch.finfo(dtype).eps / 2
    hidden = slot > held + torch.arange(rows, device="cuda")[:, None]
    for h in range(kv):
        k, v = (x[0, page, h, slot % 64].double() for x in (cache.keys, cache.values))
        z = q.reshape(rows, kv, -1, d)[:, h].double()
        p = torch.softmax((z @ k.T / d ** 0.5).masked_fill(hidden[:, None], -float("inf")), -1)
        want, size = p @ v, p @ v.abs()
        spread = (z.abs() @ k.abs().T).amax(-1, keepdim=True) / d ** 0.5
        bound = (size * (half * 1.01 + 2 * d * 2.0 ** -23 * spread + n * 2.0 ** -26 + 2.0 ** -20) + 2.0 ** -24) * (1 + half)
        assert ((got[:, h] - want).abs() <= bound + half * want.abs()).all()


def test_sequences_share_pages(kt):
    """Two sequences with the first pages in common, and tails of their own, give what copies give."""
    heads, kv, d = LLAMA
    for rows in (1, 30):
        apart = filled(LLAMA, 32, BF16, [96, 96], rows)
        shared = filled(LLAMA, 32, BF16, [96, 96], rows)
        for x in (apart, shared):
            for pool in (x.keys, x.values):
                pool[0, x.table[1, :3].long()] = pool[0, x.table[0, :3].long()]
        shared.table[1, :3] = shared.table[0, :3]
        put(apart, rows)
        put(shared, rows)
        q = queries(apart, heads, rows)
        assert torch.equal(apart.attend(0, q, heads, rows), shared.attend(0, q, heads, rows))


@pytest.mark.parametrize("layout,rows", [(LLAMA, 1), (QWEN, 70), (WIDE, 30)])
def test_attention_into_fp32_with_a_scale(kt, layout, rows):
    cache = filled(layout, 32, FP16, [90, 11], rows)
    put(cache, rows)
    q = queries(cache, layout[0], rows)
    for scale in (0.3, -0.05):
        out = torch.full((2 * rows, layout[0] * layout[2]), float("nan"), device="cuda")
        assert cache.attend(0, q, layout[0], rows, scale=scale, out=out) is out
        check_attend(cache, q, layout[0], rows, out, scale=scale)


@pytest.mark.parametrize("layout,rows", [(LLAMA, 3), (QWEN, 40), (MQA, 64)])
def test_rows_that_see_nothing_give_zeros(kt, layout, rows):
    cache = filled(layout, 16, BF16, [0, 20, 0], rows, poison=True)
    counts = torch.tensor([rows, 0, rows], dtype=torch.int32).cuda()
    put(cache, rows, counts)
    visible = torch.zeros(3, rows, (rows + 31) // 32, dtype=torch.int32, device="cuda")
    visible[2, :, 0] = 1  # all see the first token
    visible[2, 1, 0] = 0
    q = queries(cache, layout[0], rows)
    out = torch.full_like(q, float("nan"))
    cache.attend(0, q, layout[0], rows, counts, visible, out=out)
    assert not out[:2 * rows].any() and not out[2 * rows + 1].any()
    check_attend(cache, q, layout[0], rows, out, counts, visible)


@pytest.mark.parametrize("rows", [8, 70])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_seen_has_no_part(kt, rows, bad):
    """A drafted node whose key or value is not finite reaches the rows that see it alone."""
    from kotensor_b200.paged import draft_tree
    heads, kv, d = LLAMA
    parents = trees(1, rows, seed=5)
    _, visible = draft_tree(parents)
    seen = torch.from_numpy(visible).cuda()
    node = 3
    sees = torch.from_numpy((visible[0, :, 0] >> node & 1) > 0)
    for which in ("keys", "values"):
        cache = filled(LLAMA, 64, BF16, [100], rows, poison=True)
        put(cache, rows)
        good = cache.attend(0, q := queries(cache, heads, rows), heads, rows, visible=seen)
        slot = 100 + node
        getattr(cache, which)[0, int(cache.table[0, slot // 64]), :, slot % 64, 5] = bad
        got = cache.attend(0, q, heads, rows, visible=seen)
        assert torch.equal(got[~sees], good[~sees]) and torch.isfinite(got[~sees]).all()
        if which == "values" or bad != bad:
            assert torch.isnan(got[sees].reshape(-1, heads, d)).any(-1).all()


@pytest.mark.parametrize("layout,rows", [(QWEN, 1), (LLAMA, 40)])
def test_slots_without_a_page_are_not_seen(kt, layout, rows):
    cache = filled(layout, 16, BF16, [150, 37], rows)
    put(cache, rows)
    cache.table[0, 2] = -1
    cache.table[0, 4] = cache.pages
    cache.table[1, 0] = 2 ** 31 - 1
    q = queries(cache, layout[0], rows)
    check_attend(cache, q, layout[0], rows, cache.attend(0, q, layout[0], rows))


@pytest.mark.parametrize("layout,rows", [(QWEN, 1), (LLAMA, 3), (MHA, 60)])
def test_rows_apart_and_off_their_alignment(kt, layout, rows):
    heads, _, d = layout
    cache = filled(layout, 32, FP16, [45, 70], rows)
    put(cache, rows)
    wide = torch.zeros(2 * rows, heads * d + 5, dtype=FP16, device="cuda")
    q = queries(cache, heads, rows)
    want = cache.attend(0, q, heads, rows)
    for first in (1, 2):
        part = wide[:, first:first + heads * d]
        part.copy_(q)
        room = torch.zeros(2 * rows * heads * d + 3, dtype=FP16, device="cuda")
        out = room[first:first + 2 * rows * heads * d].view(2 * rows, heads * d)
        cache.attend(0, part, heads, rows, out=out)
        assert torch.equal(out, want) and not room[:first].any() and not room[first + out.numel():].any()


def test_offsets_past_32_bits(kt):
    """The last page of the last layer lies 2^32 elements behind the first."""
    from kotensor_b200.paged import PagedKVCache
    cache = PagedKVCache(layers=9, batch=1, kv_heads=8, head_dim=128, pages=8200, max_tokens=200, page=64, dtype=BF16)
    assert cache.keys.numel() > 1 << 32
    cache.table[0] = torch.tensor([8199, 8197, 8198, 8196], dtype=torch.int32)
    cache.lengths[0] = 130
    for layer in (0, 8):
        cache.keys[layer, 8190:].normal_()
        cache.values[layer, 8190:].normal_()
    for rows in (1, 40):
        put(cache, rows, layer=8)
        q = queries(cache, 32, rows)
        got = cache.attend(8, q, 32, rows)
        small = filled(LLAMA, 64, BF16, [130], 70, spare=1)
        small.table[0] = torch.tensor([3, 1, 2, 0], dtype=torch.int32)
        small.keys[0, :4], small.values[0, :4] = cache.keys[8, 8196:], cache.values[8, 8196:]
        assert torch.equal(got, small.attend(0, q, 32, rows))
        check_attend(small, q, 32, rows, got)
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32).cuda()
    before = cache.keys[8, 8198].clone()
    cache.accept(torch.tensor([[1, 2, 3]], dtype=torch.int32).cuda(), parents, torch.tensor([[3, 0, 0]], dtype=torch.int32).cuda())
    assert torch.equal(cache.keys[8, 8198, :, 3], before[:, 4])


# ---------------------------------------------------------------- accept

@pytest.mark.parametrize("layout,page,lengths,rows,dtype", [
    (QWEN, 16, [0], 1, BF16), (LLAMA, 64, [63, 100, 0], 24, BF16), (ODD, 32, [31, 5], 61, FP16), (WIDE, 128, [500, 2, 128, 127], 40, FP16),
    (MHA, 16, [14], 300, BF16),
])
@pytest.mark.parametrize("ragged", [False, True])
def test_accepted_path(kt, layout, page, lengths, rows, dtype, ragged):
    from oracle import paged_oracle as PO
    rng = np.random.default_rng(rows)
    batch = len(lengths)
    cache = filled(layout, page, dtype, lengths, rows, layers=3)
    parents = trees(batch, rows, seed=rows)
    tokens = rng.integers(0, 3, (batch, rows))  # siblings often have the same token
    choices = rng.integers(0, 3, (batch, rows))
    counts = np.array([max(0, rows - 5 * i - 1) for i in range(batch)]) if ragged else np.full(batch, rows)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).int().cuda()  # noqa: E731
    want = [x.clone().cpu() for x in (cache.keys, cache.values)]
    kept = cache.lengths.clone()
    accepted, taken = cache.accept(dev(tokens), dev(parents), dev(choices), dev(counts) if ragged else None)
    lens = []
    for b, held in enumerate(lengths):
        nodes = PO.path(tokens[b], parents[b], choices[b], int(counts[b]))
        lens.append(len(nodes))
        where = PO.slots(cache.table.cpu(), b, held + rows, page, cache.pages)[held:]
        for x in want:
            moved = [x[:, where[u][0], :, where[u][1]].clone() for u in nodes]
            for (p, i), y in zip(where, moved):
                x[:, p, :, i] = y
        assert accepted[b].tolist() == [int(choices[b][u]) for u in nodes] + [-1] * (rows - len(nodes))
    assert taken.tolist() == lens
    assert torch.equal(cache.keys.cpu(), want[0]) and torch.equal(cache.values.cpu(), want[1])
    assert torch.equal(cache.lengths, kept) and int(cache.status) == 0
    cache.advance(rows, counts=taken)
    assert cache.lengths.tolist() == [n + m for n, m in zip(lengths, lens)]


def test_a_long_path_moves_over_pages(kt):
    """Every node agrees: the path goes through lowest children to a leaf, far behind its place."""
    from oracle import paged_oracle as PO
    rows = 200
    cache = filled(QWEN, 16, FP16, [13], rows, layers=2)
    parents = np.arange(rows) - 3  # three chains from node 0
    parents[:3] = [-1, 0, 0]
    nodes = PO.path(np.ones(rows), parents, np.ones(rows), rows)
    assert len(nodes) > 60 and nodes[-1] > 190
    where = PO.slots(cache.table.cpu(), 0, 13 + rows, 16, cache.pages)[13:]
    want = cache.keys.clone()
    for i, u in enumerate(nodes):
        want[:, where[i][0], :, where[i][1]] = cache.keys[:, where[u][0], :, where[u][1]]
    ones = torch.ones(1, rows, dtype=torch.int32, device="cuda")
    _, taken = cache.accept(ones, torch.from_numpy(parents).int()[None].cuda(), ones)
    assert taken.tolist() == [len(nodes)] and torch.equal(cache.keys, want)


def test_accept_ignores_what_is_no_tree(kt):
    """Parents that are no earlier node lead nowhere; the walk ends."""
    cache = filled(QWEN, 16, BF16, [3, 3], 6)
    parents = torch.tensor([[0, 1, 5, 0, 9, -7], [-1, 0, 1, 2, 3, 4]], dtype=torch.int32).cuda()
    same = torch.ones(2, 6, dtype=torch.int32, device="cuda")
    accepted, taken = cache.accept(same, parents, same)
    assert taken.tolist() == [2, 6] and accepted.tolist() == [[1, 1, -1, -1, -1, -1], [1] * 6]


# ---------------------------------------------------------------- used together

def test_a_verified_tree_continues_as_plain_steps_do(kt):
    """Append a tree, attend, accept, go on: the cache and the attention are those of the
    accepted tokens fed one by one."""
    heads, kv, d = LLAMA
    gen = torch.Generator().manual_seed(11)
    parents = np.array([[-1, 0, 0, 1, 2, 2, 5], [-1, 0, 1, 2, 0, 4, 5]])
    tokens = torch.tensor([[9, 1, 2, 3, 4, 5, 6], [9, 1, 2, 3, 4, 5, 6]], dtype=torch.int32).cuda()
    choices = torch.tensor([[2, 0, 5, 0, 0, 6, 8], [1, 2, 7, 0, 0, 0, 0]], dtype=torch.int32).cuda()
    nodes = [[0, 2, 5, 6], [0, 1, 2]]
    from kotensor_b200.paged import draft_tree
    depths, visible = (torch.from_numpy(x).cuda() for x in draft_tree(parents))
    rows = parents.shape[1]
    x = torch.randn(2, rows, (heads + 2 * kv) * d, generator=gen).cuda()
    inv_freq = (500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().cuda()

    def feed(cache, part, **how):
        q, k, v = part.reshape(-1, part.shape[-1]).split([heads * d, kv * d, kv * d], 1)
        n = part.shape[1]
        q = cache.append(0, q, k, v, inv_freq, n, depths=how.get("depths"))
        return cache.attend(0, q, heads, n, visible=how.get("visible")).reshape(cache.batch, n, -1)

    tree = filled(LLAMA, 16, BF16, [61, 7], 12)
    out = feed(tree, x, depths=depths, visible=visible)
    accepted, taken = tree.accept(tokens, torch.from_numpy(parents).int().cuda(), choices)
    assert taken.tolist() == [4, 3] and accepted[0].tolist() == [2, 5, 6, 8, -1, -1, -1]
    tree.advance(rows, counts=taken)
    for b in range(2):
        plain = filled(LLAMA, 16, BF16, [61, 7], 12)
        one = plain.sequences(b, b + 1)
        for i, u in enumerate(nodes[b]):
            got = feed(one, x[b:b + 1, u:u + 1])
            assert torch.allclose(got[0, 0].float(), out[b, u].float(), rtol=2 ** -7, atol=2 ** -7 * float(out.abs().max()))
            one.advance(1)
        last = torch.randn(1, 1, x.shape[-1], generator=gen).cuda()
        view = tree.sequences(b, b + 1)
        assert torch.equal(feed(view, last), feed(one, last))
        assert tree.lengths[b] == plain.lengths[b]


def test_prompt_in_chunks_equals_the_whole(kt):
    heads, kv, d = QWEN
    whole, parts = (filled(QWEN, 64, FP16, [0, 0], 200) for _ in range(2))
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(2, 180, (heads + 2 * kv) * d, generator=gen).cuda()
    inv_freq = torch.rand(d // 2, generator=gen).cuda()

    def feed(cache, part):
        n = part.shape[1]
        q, k, v = part.reshape(-1, part.shape[-1]).split([heads * d, kv * d, kv * d], 1)
        got = cache.attend(0, cache.append(0, q, k, v, inv_freq, n), heads, n)
        cache.advance(n)
        return got.reshape(2, n, -1)

    want = feed(whole, x)
    got = torch.cat([feed(parts, part) for part in x.split([1, 77, 33, 69], 1)], 1)
    assert torch.equal(whole.keys, parts.keys) and torch.equal(whole.values, parts.values)
    # two results of the same sums in other orders, each within half a step twice over (probability, result)
    assert ((got.double() - want.double()).abs() <= 2 ** -10 * (want.double().abs() + want.abs().amax().double())).all()


def test_equal_bits_on_streams_and_in_replays(kt):
    heads, kv, d = LLAMA
    for rows, lengths in ((1, [3000, 17, 900]), (40, [700, 0, 1300])):
        cache = filled(LLAMA, 64, BF16, lengths, rows + 8)
        put(cache, rows)
        q = queries(cache, heads, rows)
        want = cache.attend(0, q, heads, rows)
        assert all(torch.equal(cache.attend(0, q, heads, rows), want) for _ in range(5))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            out = cache.attend(0, q, heads, rows)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        # a captured call replays at other lengths and tables, in turn with another graph and eager calls
        graphs, outs = [], []
        for _ in range(2):
            g, o = torch.cuda.CUDAGraph(), torch.empty_like(q)
            with torch.cuda.graph(g):
                cache.attend(0, q, heads, rows, out=o)
            graphs.append(g), outs.append(o)
        for shift in (0, -5, 8):
            cache.lengths.copy_(torch.tensor([max(0, n + shift) for n in lengths], dtype=torch.int32))
            cache.table.copy_(cache.table.flip(0))
            now = cache.attend(0, q, heads, rows)
            for g, o in zip(graphs, outs):
                g.replay()
                assert torch.equal(o, now)
        assert not cache.scratch[:4096].any()


def test_pages_are_handed_out_and_come_back(kt):
    from kotensor_b200.paged import PagedKVCache
    cache = PagedKVCache(1, 2, 2, 64, pages=5, max_tokens=100, page=32)
    cache.reserve(0, 33)
    cache.reserve(1, 1)
    assert cache.free_pages == 2 and (cache.table >= 0).sum(1).tolist() == [2, 1]
    cache.reserve(0, 40)
    assert cache.free_pages == 2
    with pytest.raises(ValueError, match="3 pages wanted, 2 are free"):
        cache.reserve(1, 100)
    with pytest.raises(ValueError, match="do not fit"):
        cache.reserve(1, 129)
    cache.lengths.fill_(20)
    cache.release(0)
    assert cache.free_pages == 4 and cache.table[0].tolist() == [-1] * 4 and cache.lengths.tolist() == [0, 20]
    cache.sequences(1, 2).reserve(0, 100)
    assert cache.free_pages == 1 and (cache.table[1] >= 0).all()
    assert len(set(cache.table[1].tolist())) == 4


def test_no_rows(kt):
    cache = filled(QWEN, 16, BF16, [5], 4)
    empty = torch.empty(0, 2 * 64, device="cuda")
    cache.append(0, None, empty, empty, torch.zeros(32, device="cuda"), 0)
    assert cache.attend(0, torch.empty(0, 14 * 64, dtype=BF16, device="cuda"), 14, 0).shape == (0, 14 * 64)
