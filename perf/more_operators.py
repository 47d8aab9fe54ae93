"""A paged 16-bit key/value cache, measured one pass at a time: appending rotated keys and values, attention of single
tokens, drafted trees and prompts over the pages, and the acceptance of a path of a drafted tree.

`run` computes an operator either in its plain form (elementary torch operations in 32 bits, angles in 64) or, where
`own` is true, by the calls that a user makes of kotensor_b200.  Both work on the same buffers, made by `prepare`.

The cache holds, for each layer, `pages` pages of `page` slots of every key/value head: [pages, kv, page, dim].  Slot s of
sequence b is slot s % page of page table[b][s // page].  Row t of a call is the token in slot lengths[b] + t.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one more token for each of 64 sequences of the Llama-3-8B shape, at any place inside a page
        dict(name="append token x64", op="append", batch=64, rows=1, heads=32, kv=8, dim=128, page=64, type="bf16",
             shortest=37, longest=4095, tree=False, ragged=False),
        # two drafted trees of the Qwen2-0.5B shape far into a text: angles of far positions, some rows unused
        dict(name="append tree 2x61 far", op="append", batch=2, rows=61, heads=14, kv=2, dim=64, page=16, type="fp16",
             shortest=70001, longest=100003, tree=True, ragged=True),
        # four prompts of odd length, some after earlier turns
        dict(name="append prompt 4x1021", op="append", batch=4, rows=1021, heads=32, kv=8, dim=128, page=32, type="bf16",
             shortest=0, longest=1000, tree=False, ragged=False),
        # one decode step of the Qwen2-0.5B shape early in an answer: latency is all
        dict(name="attend 1x301 hd64", op="attend", batch=1, rows=1, heads=14, kv=2, dim=64, page=16, type="fp16",
             shortest=300, longest=300, tree=False, ragged=False),
        # a full server: 64 ragged sequences of the Llama-3-8B shape, one token each
        dict(name="attend 64 ragged 8k", op="attend", batch=64, rows=1, heads=32, kv=8, dim=128, page=64, type="bf16",
             shortest=3001, longest=8190, tree=False, ragged=False),
        # one sequence with a long context: the split over slots has to fill the card
        dict(name="attend 1x120001", op="attend", batch=1, rows=1, heads=32, kv=8, dim=128, page=64, type="bf16",
             shortest=120000, longest=120000, tree=False, ragged=False),
        # drafted trees of a few requests over long contexts
        dict(name="attend tree 4x63 over 6k", op="attend", batch=4, rows=63, heads=32, kv=8, dim=128, page=32, type="bf16",
             shortest=2500, longest=6001, tree=True, ragged=False),
        # small drafted trees of a ragged batch, not all rows in use
        dict(name="attend tree 16x33 ragged", op="attend", batch=16, rows=33, heads=14, kv=2, dim=64, page=64, type="fp16",
             shortest=100, longest=4095, tree=True, ragged=True),
        # a chunk of two prompts over what the cache already holds
        dict(name="attend chunk 2x509", op="attend", batch=2, rows=509, heads=32, kv=8, dim=128, page=64, type="bf16",
             shortest=1000, longest=2999, tree=False, ragged=False),
        # a whole prompt into an empty cache
        dict(name="attend prompt 1x4093", op="attend", batch=1, rows=4093, heads=32, kv=8, dim=128, page=128, type="bf16",
             shortest=0, longest=0, tree=False, ragged=False),
        # the tree of one request of the Qwen2-0.5B shape is checked: latency is all
        dict(name="accept 1x24", op="accept", batch=1, rows=24, layers=24, kv=2, dim=64, page=64, type="bf16",
             shortest=50, longest=50, depth=6, ragged=False),
        # the trees of 16 requests of the Llama-3-8B shape
        dict(name="accept 16x61", op="accept", batch=16, rows=61, layers=32, kv=8, dim=128, page=32, type="bf16",
             shortest=3, longest=60, depth=9, ragged=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "accept"])
    heads, kv, dim = rng.choice([(14, 2, 64), (32, 8, 128), (12, 12, 64), (8, 1, 128), (15, 5, 80), (24, 2, 96)])
    c = dict(op=op, heads=heads, kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128]), type=rng.choice(["bf16", "fp16"]))
    if op == "append":
        c["tree"] = rng.random() < 0.4
        c["rows"] = rows = _log(rng, 2, 100) if c["tree"] else rng.choice([1, _log(rng, 2, 1021)])
        longest = _log(rng, 1, 100000 if rng.random() < 0.3 else 4000)
        room = 64 * 4200 * 8 * 128 // ((longest + rows) * kv * dim)
        c["batch"] = max(1, min(_log(rng, 1, 128 if rows == 1 else 16), room, 4 * 1021 * 40 * 128 // (rows * (heads + kv) * dim)))
    elif op == "attend":
        kind = rng.choice(["token", "tree", "chunk"])
        c["tree"] = kind == "tree"
        c["rows"] = rows = 1 if kind == "token" else _log(rng, 2, 100) if c["tree"] else _log(rng, 2, 2000)
        longest = _log(rng, 1, 100000 if rows == 1 else 20000 if c["tree"] else 2000)
        room = 64 * 5500 * 8 * 128 // ((longest + rows) * kv * dim)
        work = 4093 * 4093 * 32 * 128 // (2 * rows * (longest + rows) * heads * dim)
        c["batch"] = max(1, min(_log(rng, 1, 64), room, work if rows > 1 else room))
    else:
        del c["heads"]
        c["rows"] = rows = _log(rng, 2, 100)
        c["depth"] = rng.randint(1, min(12, rows - 1))
        c["layers"] = rng.choice([2, 24, 32])
        longest = _log(rng, 1, 100)
        c["batch"] = max(1, min(_log(rng, 1, 64), 16 * 130 * 32 * 8 * 128 // ((longest + rows + 20) * c["layers"] * kv * dim)))
    return c | dict(shortest=rng.randint(0, longest), longest=longest, ragged=rng.random() < 0.5 and c["rows"] > 1)


def _lengths(c):
    """Tokens held by each sequence, the same for every seed: spread from `shortest` to `longest`, out of order."""
    b, low, high = c["batch"], c["shortest"], c["longest"]
    return [high] if b == 1 else [low + (high - low) * ((i * 7 + 3) % b) // (b - 1) for i in range(b)]


def _counts(c):
    """Rows in use of each sequence: all, or fewer in some."""
    return [c["rows"] - (c["rows"] * (i % 4) // 5 if c["ragged"] else 0) for i in range(c["batch"])]


def _trees(c):
    """Parents [batch, rows] of drafted trees, the same for every seed: node 0 is the last token of the text, a third of
    the nodes go on from the node before them (chains) and the others from one of the first (branches)."""
    deepest = c.get("depth", 8)
    every = []
    for b in range(c["batch"]):
        parents, depth = [-1], [0]
        for i in range(1, c["rows"]):
            p = i - 1 if (i * 5 + b) % 3 else (i * 13 + b * 7) % i
            while depth[p] >= deepest:
                p = parents[p]
            parents.append(p)
            depth.append(depth[p] + 1)
        every.append(parents)
    return every


def _levels(parents):
    """(depths, whether u is t or above it) of each tree."""
    depths, above = [], []
    for tree in parents:
        d, a = [], []
        for t, p in enumerate(tree):
            line = [False] * len(tree) if p < 0 else list(a[p])
            line[t] = True
            d.append(0 if p < 0 else d[p] + 1)
            a.append(line)
        depths.append(d)
        above.append(a)
    return depths, above


# ---------------------------------------------------------------- what a program has in hand

def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype = TYPES[c["type"]]
    b, rows, kv, d, page = c["batch"], c["rows"], c["kv"], c["dim"], c["page"]
    layers = c.get("layers", 1)
    width = -(-(c["longest"] + rows) // page)  # pages of a sequence
    pool = b * width + 3
    s = {"case": c}
    # keys with channels of unequal size and a common offset, as rotary keys have them, values without
    gain = torch.exp(0.5 * torch.randn(kv, 1, d, generator=gen, device=dev))
    offset = 0.5 * torch.randn(kv, 1, d, generator=gen, device=dev)
    for name in ("keys", "values"):
        x = torch.empty(layers, pool, kv, page, d, dtype=dtype, device=dev)
        step = max(1, (1 << 28) // (kv * page * d))
        for l in range(layers):
            for i in range(0, pool, step):
                part = torch.randn(min(step, pool - i), kv, page, d, generator=gen, device=dev)
                x[l, i:i + step] = part * gain + offset if name == "keys" else part
        s[name] = x
    s["table"] = torch.randperm(pool, generator=gen, device=dev)[:b * width].reshape(b, width).int()
    s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=dev)
    s["counts"] = torch.tensor(_counts(c), dtype=torch.int32, device=dev) if c["ragged"] else None
    s["depths"] = s["visible"] = None
    if c["op"] == "accept":
        trees = _trees(c)
        s["parents"] = torch.tensor(trees, dtype=torch.int32, device=dev)
        s["tokens"] = torch.randint(0, 128256, (b, rows), generator=gen, device=dev).int()
        # three of four nodes that have children choose one of them
        choices = torch.randint(0, 128256, (b, rows), generator=gen, device=dev).int()
        lucky = (torch.rand(b, rows, generator=gen, device=dev) < 0.75).tolist()
        pick = torch.rand(b, rows, generator=gen, device=dev).tolist()
        held = s["tokens"].tolist()
        chosen = choices.tolist()
        for i, tree in enumerate(trees):
            children = [[] for _ in tree]
            for t, p in enumerate(tree):
                if p >= 0:
                    children[p].append(t)
            for t, below in enumerate(children):
                if below and lucky[i][t]:
                    chosen[i][t] = held[i][below[int(pick[i][t] * len(below))]]
        s["choices"] = torch.tensor(chosen, dtype=torch.int32, device=dev)
    else:
        if c["tree"]:
            depths, above = _levels(_trees(c))
            s["depths"] = torch.tensor(depths, dtype=torch.int32, device=dev)
            words = -(-rows // 32)
            bits = torch.zeros(b, rows, words * 32, dtype=torch.int64, device=dev)
            bits[:, :, :rows] = torch.tensor(above, dtype=torch.int64, device=dev)
            word = (bits.reshape(b, rows, words, 32) << torch.arange(32, device=dev)).sum(-1)
            s["visible"] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()
        if c["op"] == "append":
            fused = torch.randn(b * rows, (c["heads"] + 2 * kv) * d, generator=gen, device=dev)  # as the projection leaves it
            fused[:, c["heads"] * d:(c["heads"] + kv) * d] *= gain.expand(kv, 1, d).reshape(-1)
            s["q"], s["k"], s["v"] = fused.split([c["heads"] * d, kv * d, kv * d], 1)
            exponent = torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d
            s["inv_freq"] = (500000.0 ** -exponent).float()
            s["q_out"] = torch.zeros(b * rows, c["heads"] * d, dtype=dtype, device=dev)
        else:
            s["q"] = (2.0 * torch.randn(b * rows, c["heads"] * d, generator=gen, device=dev)).to(dtype)
            s["out"] = torch.empty(b * rows, c["heads"] * d, dtype=dtype, device=dev)
    if own:
        from kotensor_b200.paged import PagedKVCache
        cache = PagedKVCache(layers=layers, batch=b, kv_heads=kv, head_dim=d, pages=pool, max_tokens=width * page, page=page,
                             dtype=dtype)
        for name in ("keys", "values", "table", "lengths"):
            getattr(cache, name).copy_(s[name])
            s[name] = getattr(cache, name)
        s["cache"] = cache
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    if c["op"] == "append":
        if own:
            s["cache"].append(0, s["q"], s["k"], s["v"], s["inv_freq"], rows_per_seq=c["rows"], counts=s["counts"],
                              depths=s["depths"], out=s["q_out"])
        else:
            _plain_append(s)
        return {"q": s["q_out"], "keys": s["keys"], "values": s["values"]}
    if c["op"] == "attend":
        if own:
            s["cache"].attend(0, s["q"], c["heads"], rows_per_seq=c["rows"], counts=s["counts"], visible=s["visible"],
                              out=s["out"])
        else:
            _plain_attend(s)
        return {"out": s["out"]}
    if own:
        accepted, taken = s["cache"].accept(s["tokens"], s["parents"], s["choices"], counts=s["counts"])
    else:
        accepted, taken = _plain_accept(s)
    return {"accepted": accepted, "taken": taken, "keys": s["keys"], "values": s["values"]}


def _rows_in_use(s):
    """[batch, rows]: whether a row is a token."""
    c = s["case"]
    t = torch.arange(c["rows"], device=s["lengths"].device).expand(c["batch"], c["rows"])
    return t < (c["rows"] if s["counts"] is None else s["counts"][:, None])


def _places(s, slot):
    """(page, slot in it) of slots [batch, n]."""
    page = s["case"]["page"]
    return s["table"].long().gather(1, (slot // page).clamp(max=s["table"].shape[1] - 1)), slot % page


def _plain_append(s):
    """Queries and keys turned by their positions' angles, pairs half a head apart; keys and values into the pages, queries
    into rows of the cache's type.  Rows that are no tokens give zeros and store nothing."""
    c = s["case"]
    b, t, d = c["batch"], c["rows"], c["dim"]
    row = torch.arange(t, device=s["q"].device).expand(b, t)
    used = _rows_in_use(s)
    at = s["lengths"].long()[:, None] + (row if s["depths"] is None else s["depths"])
    angle = at[:, :, None].double() * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]

    def turned(x):
        x = x.reshape(b, t, -1, d)
        low, high = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([low * cos - high * sin, low * sin + high * cos], -1)

    dtype = s["keys"].dtype
    s["q_out"].copy_((turned(s["q"]) * used[:, :, None, None]).reshape(b * t, -1).to(dtype))
    place, slot = _places(s, s["lengths"].long()[:, None] + row)
    if s["counts"] is not None:  # rows that are no tokens write what the last one does
        last = (s["counts"].long() - 1)[:, None]
        pick = torch.minimum(row, last)
        place, slot = place.gather(1, pick), slot.gather(1, pick)
        pick = pick[:, :, None, None]
    else:
        pick = row[:, :, None, None]
    for name, x in (("keys", turned(s["k"])), ("values", s["v"].reshape(b, t, -1, d))):
        x = x.gather(1, pick.expand(x.shape)).to(dtype)
        s[name][0].transpose(1, 2)[place, slot] = x


def _plain_attend(s):
    """Softmax of the scores of what a row sees times the values; the heads of a group share keys and values.  Rows that
    are no tokens give zeros."""
    c = s["case"]
    b, kv, d, t, h, page = c["batch"], c["kv"], c["dim"], c["rows"], c["heads"], c["page"]
    group, dev = h // kv, s["q"].device
    span = s["table"].shape[1] * page
    slot = torch.arange(span, device=dev)
    new = slot - s["lengths"][:, None]  # [b, span]: which row of the call is in a slot
    row = torch.arange(t, device=dev)
    if s["visible"] is None:
        seen = new[:, None] <= row[:, None]
    else:
        bits = ((s["visible"][..., None] >> torch.arange(32, device=dev)) & 1).reshape(b, t, -1)[..., :t] > 0
        seen = bits.gather(2, new.clamp(0, t - 1)[:, None].expand(b, t, span)) & (new < t)[:, None]
        seen = seen | (new < 0)[:, None]
    used = _rows_in_use(s)
    seen = seen & (new < used.sum(1, keepdim=True))[:, None] & used[:, :, None]
    out = s["out"].reshape(b, t, kv, group, d)
    step = max(1, (1 << 31) // max(span * kv * d, h * t * span))  # sequences at a time
    for i in range(0, b, step):
        n = min(step, b - i)
        pages = s["table"][i:i + n].long()
        k, v = (s[x][0][pages].transpose(1, 2).reshape(n, kv, span, d).float() for x in ("keys", "values"))
        q = s["q"][i * t:(i + n) * t].float().reshape(n, t, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n, kv, group * t, d)
        score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
        del k
        mask = seen[i:i + n, None, None]
        score = score.reshape(n, kv, group, t, span).masked_fill_(~mask, -math.inf)
        top = score.amax(-1, keepdim=True)
        p = torch.exp_(score - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        y = torch.matmul(p.reshape(n, kv, group * t, span), v).reshape(n, kv, group, t, d)
        y = y / torch.where(total == 0, 1.0, total)
        out[i:i + n] = y.permute(0, 3, 1, 2, 4).to(s["out"].dtype)


def _plain_accept(s):
    """From node 0 on, the lowest child whose token is its parent's choice; the path's keys and values move to the slots
    behind the text, and the choices along it are the new tokens."""
    c = s["case"]
    b, rows = c["batch"], c["rows"]
    dev = s["tokens"].device
    node = torch.arange(rows, device=dev).expand(b, rows)
    used = _rows_in_use(s)
    at = torch.zeros(b, dtype=torch.int64, device=dev)
    going = used[:, 0]
    path = node.clone()  # nodes behind the path's end stay where they are
    taken = going.int()
    accepted = torch.full((b, rows), -1, dtype=torch.int32, device=dev)
    accepted[:, 0] = torch.where(going, s["choices"][:, 0], -1)
    for i in range(1, c["depth"] + 1):
        choice = s["choices"].gather(1, at[:, None])
        fits = (s["parents"] == at[:, None]) & (s["tokens"] == choice) & used & (node > at[:, None])
        nearest = torch.where(fits, node, rows).amin(1)
        going = going & (nearest < rows)
        at = torch.where(going, nearest, at)
        path[:, i] = torch.where(going, at, path[:, i])
        taken = taken + going.int()
        accepted[:, i] = torch.where(going, s["choices"].gather(1, at[:, None])[:, 0], -1)
    move = c["depth"] + 1
    held = s["lengths"].long()[:, None]
    source, target = _places(s, held + path[:, :move]), _places(s, held + node[:, :move])
    for name in ("keys", "values"):
        x = s[name].transpose(2, 3)  # [layers, pages, page, kv, dim]
        x[:, target[0], target[1]] = x[:, source[0], source[1]]
    return accepted, taken


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    kv, d, held, counts = c["kv"], c["dim"], _lengths(c), _counts(c)
    if c["op"] == "append":
        width = (c["heads"] + 2 * kv) * d
        return {"bytes": sum(counts) * width * 6 + 2 * (c["batch"] * c["rows"] - sum(counts)) * c["heads"] * d,
                "flops": 6 * sum(counts) * width}
    if c["op"] == "attend":
        slots = sum(n + m for n, m in zip(held, counts))
        if c["tree"]:
            _, above = _levels(_trees(c))
            new = sum(sum(map(sum, (line[:m] for line in tree[:m]))) for tree, m in zip(above, counts))
        else:
            new = sum(m * (m + 1) // 2 for m in counts)
        pairs = new + sum(n * m for n, m in zip(held, counts))
        rows = c["batch"] * c["rows"] + sum(counts)
        return {"bytes": 4 * kv * d * slots + 2 * rows * c["heads"] * d, "flops": 4 * pairs * c["heads"] * d}
    # a path of about half the depth, of which all but the first token move
    moved = c["batch"] * max(1, c["depth"] // 2)
    return {"bytes": 8 * kv * d * c["layers"] * moved + 16 * c["batch"] * c["rows"], "flops": 2 * c["batch"] * c["rows"]}


# ---------------------------------------------------------------- the same in 64 bits, written apart

def exact(case, seed):
    """What `run` returns, in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "attend": _exact_attend, "accept": _exact_accept}[case["op"]](s)


def _slots(s, b, n):
    """(pages, places in them) of the first n slots of sequence b."""
    page = s["case"]["page"]
    at = torch.arange(n, device=s["table"].device)
    return s["table"][b].long()[at // page], at % page


def _exact_append(s):
    c = s["case"]
    t, d, half = c["rows"], c["dim"], c["dim"] // 2
    keys, values = s["keys"].double(), s["values"].double()
    q = torch.zeros(c["batch"], t, c["heads"], d, dtype=torch.float64, device=s["q"].device)
    for b, (n, m) in enumerate(zip(_lengths(c), _counts(c))):
        where = torch.arange(m, device=q.device) if s["depths"] is None else s["depths"][b, :m]
        angle = torch.outer((n + where).double(), s["inv_freq"].double())[:, None]
        turn = torch.polar(torch.ones_like(angle), angle)
        lines = slice(b * t, b * t + m)
        for source, target in ((s["q"], q[b, :m]), (s["k"], None)):
            x = source[lines].double().reshape(m, -1, 2, half)
            z = torch.complex(x[:, :, 0].contiguous(), x[:, :, 1].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
            if target is not None:
                target.copy_(y)
        page, place = (x[n:] for x in _slots(s, b, n + m))
        for i in range(m):
            keys[0, page[i], :, place[i]] = y[i]
            values[0, page[i], :, place[i]] = s["v"][b * t + i].double().reshape(-1, d)
    return {"q": q.reshape(c["batch"] * t, -1), "keys": keys, "values": values}


def _exact_attend(s):
    c = s["case"]
    t, d, kv, h = c["rows"], c["dim"], c["kv"], c["heads"]
    out = torch.zeros(c["batch"], t, kv, h // kv, d, dtype=torch.float64, device=s["q"].device)
    above = _levels(_trees(c))[1] if c["tree"] else None
    for b, (n, m) in enumerate(zip(_lengths(c), _counts(c))):
        page, place = _slots(s, b, n + m)
        q = s["q"].reshape(c["batch"], t, kv, -1, d)[b, :m].double()
        new = torch.ones(m, m, device=q.device).tril() if above is None else torch.tensor(above[b], device=q.device)[:m, :m]
        hidden = torch.cat([torch.zeros(m, n, dtype=torch.bool, device=q.device), new == 0], 1)
        for i in range(kv):
            k, v = (s[x][0, page, i, place].double() for x in ("keys", "values"))
            for first in range(0, m, 1024):
                some = slice(first, min(m, first + 1024))
                z = torch.einsum("tgd,sd->gts", q[some, i], k) / math.sqrt(d)
                p = torch.softmax(z.masked_fill(hidden[some], -math.inf), -1)
                out[b, some, i] = torch.einsum("gts,sd->tgd", p, v)
    return {"out": out.reshape(c["batch"] * t, h * d)}


def _exact_accept(s):
    c = s["case"]
    accepted, taken = [], []
    keys, values = s["keys"].double(), s["values"].double()
    tokens, parents, choices = (s[x].tolist() for x in ("tokens", "parents", "choices"))
    for b, (n, m) in enumerate(zip(_lengths(c), _counts(c))):
        path = [0]
        while True:
            below = [u for u in range(path[-1] + 1, m) if parents[b][u] == path[-1] and tokens[b][u] == choices[b][path[-1]]]
            if not below:
                break
            path.append(below[0])
        page, place = _slots(s, b, n + c["rows"])
        for x in (keys, values):
            moved = [x[:, page[n + u], :, place[n + u]].clone() for u in path]
            for i, y in enumerate(moved):
                x[:, page[n + i], :, place[n + i]] = y
        taken.append(len(path))
        accepted.append([choices[b][u] for u in path] + [-1] * (c["rows"] - len(path)))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "taken": torch.tensor(taken, dtype=torch.int32),
            "keys": keys, "values": values}
