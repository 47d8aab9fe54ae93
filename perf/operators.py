"""Serving operators measured one pass at a time: the 8-bit key/value cache (store, attention, eviction) and the
processing of logits before the next token is chosen.

`run` computes an operator either in its plain form (elementary torch operations in 32 bits) or, where `own` is true,
by the calls that a user makes of kotensor_b200.  Both work on the same buffers, made by `prepare`.

The cache of one layer holds, for each sequence and key/value head, `capacity` slots of `head_dim` signed bytes and one
float32 scale for every `block` slots; the slots after the last full block (the open block) are also kept in float32
(`tail`), so that a token added to the block re-quantises the block from its original values.  For a block with largest
magnitude a:  scale = a * (1/127),  code = round_half_even(x * (127 * (1/a))), and 0 for both where a < 2^-100.
"""
import math

import torch

own = False

NEG = -1e9  # the framework's greedy rule: a logit has to be above this to be chosen, else token 0


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one more token for 64 sequences of the Llama-3-8B shape, at any place inside a block
        dict(name="store token x64", op="store", batch=64, rows=1, kv=8, dim=128, block=64, shortest=37, longest=4095),
        # the prompts of four sequences, odd length, two of them after earlier turns
        dict(name="store prompt 4x1021", op="store", batch=4, rows=1021, kv=8, dim=128, block=64, shortest=0, longest=1000),
        # one decode step of the Qwen2-0.5B shape early in an answer: latency is all
        dict(name="attend 1x301 hd64", op="attend", batch=1, rows=1, heads=14, kv=2, dim=64, block=64, shortest=300,
             longest=300, weights=False),
        # a ragged batch of the Llama-3-8B shape that also keeps the accumulated weights for eviction
        dict(name="attend 16 ragged +weights", op="attend", batch=16, rows=1, heads=32, kv=8, dim=128, block=64,
             shortest=130, longest=8190, weights=True),
        # one sequence with a long context: the split over slots has to fill the card
        dict(name="attend 1x120001", op="attend", batch=1, rows=1, heads=32, kv=8, dim=128, block=32, shortest=120000,
             longest=120000, weights=False),
        # a full server: 64 sequences of about 16k tokens
        dict(name="attend 64x16k", op="attend", batch=64, rows=1, heads=32, kv=8, dim=128, block=64, shortest=15501,
             longest=16382, weights=False),
        # a chunk of two prompts over what the cache already holds
        dict(name="attend chunk 2x509", op="attend", batch=2, rows=509, heads=32, kv=8, dim=128, block=64, shortest=1000,
             longest=2999, weights=False),
        # a small cache pruned to its heavy hitters
        dict(name="evict 1x1001 to 512", op="evict", batch=1, kv=2, dim=64, block=64, shortest=1001, longest=1001, keep=512,
             recent=128),
        # a ragged batch pruned to half
        dict(name="evict 16x8k to 4000", op="evict", batch=16, kv=8, dim=128, block=64, shortest=6001, longest=8191,
             keep=4000, recent=256),
        # one row of the Qwen2-0.5B vocabulary with penalties
        dict(name="logits 1x151936", op="logits", batch=1, vocab=151936, history=701, prompt=500, biases=20, mask=False),
        # 64 requests of the Llama-3-8B vocabulary under a grammar
        dict(name="logits 64x128256 mask", op="logits", batch=64, vocab=128256, history=4093, prompt=3001, biases=0, mask=True),
        # 256 requests with everything on
        dict(name="logits 256x151936", op="logits", batch=256, vocab=151936, history=1025, prompt=512, biases=300, mask=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "evict", "logits"])
    heads, kv, dim = rng.choice([(14, 2, 64), (32, 8, 128), (12, 12, 64), (8, 1, 128), (15, 5, 80), (24, 2, 96)])
    block = rng.choice([16, 32, 64])
    if op == "store":
        rows = rng.choice([1, _log(rng, 2, 1021)])
        batch = _log(rng, 1, 256) if rows == 1 else max(1, min(_log(rng, 1, 64), 4 * 1021 * 8 * 128 // (rows * kv * dim)))
        longest = _log(rng, 1, 4095 if batch > 64 else 8191)
        return dict(op=op, batch=batch, rows=rows, kv=kv, dim=dim, block=block, shortest=rng.randint(0, longest),
                    longest=longest)
    if op == "attend":
        rows = rng.choice([1, 1, _log(rng, 2, 600)])
        longest = _log(rng, 1, 100000 if rows == 1 else 4000)
        room = 64 * 16000 * 8 * 128 // (longest * kv * dim) if rows == 1 else 2 * 509 * 32 * 128 * 3500 // (rows * heads * dim * (longest + rows))
        batch = max(1, min(_log(rng, 1, 128), room))
        return dict(op=op, batch=batch, rows=rows, heads=heads, kv=kv, dim=dim, block=block,
                    shortest=rng.randint(0, longest), longest=longest, weights=rows == 1 and rng.random() < 0.4)
    if op == "evict":
        longest = _log(rng, 40, 30000)
        keep = rng.randint(max(2, longest // 8), max(3, longest * 3 // 4))
        batch = max(1, min(_log(rng, 1, 64), 16 * 8191 * 8 * 128 // (longest * kv * dim)))
        return dict(op=op, batch=batch, kv=kv, dim=dim, block=block, shortest=rng.randint(keep + 1, longest),
                    longest=longest, keep=keep, recent=rng.randint(0, keep))
    history = _log(rng, 1, 8191)
    return dict(op=op, batch=_log(rng, 1, 200), vocab=_log(rng, 1000, 160000), history=history,
                prompt=rng.randint(0, history), biases=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.5)


def _lengths(c):
    """Tokens held by each sequence, the same for every seed: spread from `shortest` to `longest`, out of order."""
    b, low, high = c["batch"], c["shortest"], c["longest"]
    return [high if b == 1 else low + (high - low) * ((i * 7 + 3) % b) // (b - 1) for i in range(b)] if b > 1 else [high]


def _histories(c):
    """(tokens so far, tokens of the prompt among them) of each row."""
    n = [c["history"] - (c["history"] * ((i * 5) % 11)) // 13 for i in range(c["batch"])]
    return n, [min(x, c["prompt"] - (c["prompt"] * (i % 3)) // 4) for i, x in enumerate(n)]


def _capacity(c):
    """Slots of a sequence: what is held, the new rows and room for two more blocks."""
    return -(-(c["longest"] + c.get("rows", 0)) // c["block"]) * c["block"] + 2 * c["block"]


# ---------------------------------------------------------------- quantisation in its plain form

def _quantise(x, block):
    """codes, scales of x [..., slots, dim] with `slots` a multiple of `block`."""
    y = x.reshape(*x.shape[:-2], -1, block, x.shape[-1])
    top = y.abs().amax((-1, -2))
    empty = top < 2.0 ** -100
    inverse = torch.where(empty, 0.0, top.reciprocal() * 127.0)
    codes = torch.round(y * inverse[..., None, None]).clamp(-127, 127).to(torch.int8)
    return codes.reshape(x.shape), torch.where(empty, 0.0, top * (1.0 / 127.0))


def _values(codes, scales, block):
    """The float32 values that codes [..., slots, dim] stand for."""
    y = codes.reshape(*codes.shape[:-2], -1, block, codes.shape[-1]).float() * scales[..., None, None]
    return y.reshape(codes.shape)


# ---------------------------------------------------------------- what a program has in hand

def _filled(c, gen, dev):
    """Buffers of a cache that holds the keys and values of every slot: keys with channels of unequal size and a common
    offset, as rotary keys have them, values without."""
    b, kv, d, block, cap = c["batch"], c["kv"], c["dim"], c["block"], _capacity(c)
    s = {}
    held = torch.tensor(_lengths(c), dtype=torch.int32, device=dev)
    gain = torch.exp(0.5 * torch.randn(kv, 1, d, generator=gen, device=dev))
    offset = 0.5 * torch.randn(kv, 1, d, generator=gen, device=dev)
    for name in ("k", "v"):
        codes = torch.empty(b, kv, cap, d, dtype=torch.int8, device=dev)
        scales = torch.empty(b, kv, cap // block, device=dev)
        tail = torch.zeros(b, kv, block, d, device=dev)
        first = (held // block * block).long()[:, None] + torch.arange(block, device=dev)  # slots of the open block
        step = max(1, (1 << 28) // (kv * cap * d))
        for i in range(0, b, step):
            n = min(step, b - i)
            x = torch.randn(n, kv, cap, d, generator=gen, device=dev)
            x = x * gain + offset if name == "k" else x
            codes[i:i + n], scales[i:i + n] = _quantise(x, block)
            tail[i:i + n] = x.gather(2, first[i:i + n, None, :, None].expand(n, kv, block, d))
        s[name + "_codes"], s[name + "_scales"], s[name + "_tail"] = codes, scales, tail
    s["gain"], s["offset"] = gain, offset
    s["lengths"] = held
    return s


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "logits":
        b, n = c["batch"], c["vocab"]
        held, prompt = _histories(c)
        s["logits"] = 3.0 * torch.randn(b, n, generator=gen, device=dev)
        # tokens of a text are far from uniform: a few come again and again
        u = torch.rand(b, max(1, max(held)), generator=gen, device=dev)
        s["tokens"] = (n * u ** 4).int().clamp(max=n - 1)
        s["lengths"] = torch.tensor(held, dtype=torch.int32, device=dev)
        s["prompt_lengths"] = torch.tensor(prompt, dtype=torch.int32, device=dev)
        s["repetition"] = 1.0 + 0.3 * torch.rand(b, generator=gen, device=dev)
        s["frequency"] = 0.5 * torch.rand(b, generator=gen, device=dev)
        s["presence"] = 0.5 * torch.rand(b, generator=gen, device=dev)
        s["bias_ids"] = s["bias_values"] = s["bias_counts"] = s["allowed"] = None
        if c["biases"]:
            e = c["biases"]
            start = torch.randint(0, n, (b, 1), generator=gen, device=dev)
            s["bias_ids"] = ((start + torch.arange(e, device=dev) * (n // e)) % n).int()  # unlike ids in a row
            s["bias_values"] = 2.0 * torch.randn(b, e, generator=gen, device=dev)
            s["bias_counts"] = torch.randint(0, e + 1, (b,), generator=gen, device=dev).int()
        if c["mask"]:
            word = lambda: torch.randint(-2 ** 31, 2 ** 31, (b, (n + 31) // 32), generator=gen, device=dev).int()  # noqa: E731
            s["allowed"] = word() & word() & word()
        s["out"] = torch.empty_like(s["logits"])
        if own:
            from kotensor_b200.logits import LogitsProcessor
            s["processor"] = LogitsProcessor(b, n)
        return s
    s.update(_filled(c, gen, dev))
    b, kv, d, cap = c["batch"], c["kv"], c["dim"], _capacity(c)
    s["weights"] = None
    if c["op"] == "store":
        rows = b * c["rows"]
        fused = torch.randn(rows, 2, kv, d, generator=gen, device=dev)  # keys and values as a projection leaves them
        fused[:, 0] = fused[:, 0] * s["gain"][:, 0] + s["offset"][:, 0]
        fused = fused.reshape(rows, 2 * kv * d)
        s["k"], s["v"] = fused[:, :kv * d], fused[:, kv * d:]
    elif c["op"] == "attend":
        s["q"] = torch.randn(b * c["rows"], c["heads"] * d, generator=gen, device=dev)
        if c["weights"]:
            s["weights"] = torch.rand(b, kv, cap, generator=gen, device=dev)
    else:
        # accumulated weights: heavy-tailed, with tokens that nothing looked at
        w = torch.exp(2.0 * torch.randn(b, kv, cap, generator=gen, device=dev))
        s["weights"] = torch.where(torch.rand(b, kv, cap, generator=gen, device=dev) < 0.2, 0.0, w)
    if own:
        from kotensor_b200.kv8 import KVCache8
        cache = KVCache8(layers=1, batch=b, kv_heads=kv, head_dim=d, capacity=cap, block=c["block"],
                         track_weights=s["weights"] is not None)
        for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail", "weights"):
            if s[name] is not None:
                getattr(cache, name)[0].copy_(s[name])
                s[name] = getattr(cache, name)[0]
        cache.lengths.copy_(s["lengths"])
        s["cache"] = cache
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    if c["op"] == "logits":
        token = _own_logits(s) if own else _plain_logits(s)
        return {"logits": s["out"], "token": token}
    if c["op"] == "store":
        if own:
            s["cache"].store(0, s["k"], s["v"], rows_per_seq=c["rows"])
        else:
            for name in ("k", "v"):
                _plain_store(s, name)
        names = ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail")
        return {n: s[n] for n in names}
    if c["op"] == "attend":
        if own:
            out = s["cache"].attend(0, s["q"], heads=c["heads"], rows_per_seq=c["rows"], accumulate=c["weights"])
        else:
            out = _plain_attend(s)
        return {"out": out, "weights": s["weights"]} if c["weights"] else {"out": out}
    if own:
        s["cache"].evict_layer(0, c["keep"], c["recent"])
    else:
        _plain_evict(s)
    names = ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail", "weights")
    return {n: s[n] for n in names}


def _own_logits(s):
    return s["processor"](s["logits"], out=s["out"], tokens=s["tokens"], lengths=s["lengths"],
                          prompt_lengths=s["prompt_lengths"], repetition=s["repetition"], frequency=s["frequency"],
                          presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                          bias_counts=s["bias_counts"], allowed=s["allowed"])


def _plain_store(s, name):
    """The new rows of each sequence into the slots from lengths[b] on: every block that they touch is quantised from
    float32 (the open block's earlier slots from `tail`), and what is left over at the end becomes the new `tail`."""
    c = s["case"]
    b, kv, d, block, t = c["batch"], c["kv"], c["dim"], c["block"], c["rows"]
    dev = s[name].device
    codes, scales, tail = s[name + "_codes"], s[name + "_scales"], s[name + "_tail"]
    held = s["lengths"].long()
    inside = held % block
    window = (-(-t // block) + 1) * block  # slots of the blocks that t rows can touch
    at = torch.arange(window, device=dev)
    row = at - inside[:, None]  # the new row in each slot of the window
    new = s[name].reshape(b, t, kv, d).transpose(1, 2)
    x = new.gather(2, row.clamp(0, t - 1)[:, None, :, None].expand(b, kv, window, d))
    old = tail.gather(2, at.clamp(max=block - 1)[None, None, :, None].expand(b, kv, window, d))
    real = row < t
    x = torch.where((row < 0)[:, None, :, None], old, x)
    x = torch.where(real[:, None, :, None], x, 0.0)
    got, scale = _quantise(x, block)
    slot = (held - inside)[:, None] + at
    place = slot.clamp(max=codes.shape[2] - 1)[:, None, :, None].expand(b, kv, window, d)
    codes.scatter_(2, place, torch.where(real[:, None, :, None], got, codes.gather(2, place)))
    group = ((held // block)[:, None] + torch.arange(window // block, device=dev)).clamp(max=scales.shape[2] - 1)
    group = group[:, None].expand(b, kv, window // block)
    touched = real.reshape(b, -1, block)[..., 0][:, None]
    scales.scatter_(2, group, torch.where(touched, scale, scales.gather(2, group)))
    end = held + t
    first = end // block * block - (held - inside)  # the new open block's place in the window
    place = (first[:, None] + torch.arange(block, device=dev)).clamp(max=window - 1)[:, None, :, None].expand(b, kv, block, d)
    kept = torch.arange(block, device=dev) < (end % block)[:, None]
    tail.copy_(torch.where(kept[:, None, :, None], x.gather(2, place), tail))


def _plain_attend(s):
    """Row t of sequence b over the slots 0 .. lengths[b] + t: softmax(q k / sqrt(dim)) v, the heads of a group sharing
    their keys and values; the weights of all rows and heads of a group are added to `weights`."""
    c = s["case"]
    b, kv, d, block, t, h = c["batch"], c["kv"], c["dim"], c["block"], c["rows"], c["heads"]
    group = h // kv
    span = -(-(c["longest"] + t) // block) * block
    k = _values(s["k_codes"][:, :, :span], s["k_scales"][:, :, :span // block], block)
    q = s["q"].reshape(b, t, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, kv, group * t, d)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    del k
    last = s["lengths"][:, None] + torch.arange(t, device=q.device)
    seen = torch.arange(span, device=q.device) <= last[:, :, None]  # [b, t, span]
    score = score.reshape(b, kv, group, t, span).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp_(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    if s["weights"] is not None:
        s["weights"][:, :, :span] += p.sum((2, 3))
    v = _values(s["v_codes"][:, :, :span], s["v_scales"][:, :, :span // block], block)
    out = torch.matmul(p.reshape(b, kv, group * t, span), v)
    return out.reshape(b, kv, group, t, d).permute(0, 3, 1, 2, 4).reshape(b * t, h * d)


def _plain_evict(s):
    """Each head keeps its `recent` last slots and, of the others, those of the largest accumulated weight (the lowest
    slot among equal ones), in their order; the kept values are quantised again in their new blocks."""
    c = s["case"]
    b, kv, d, block, keep = c["batch"], c["kv"], c["dim"], c["block"], c["keep"]
    w = s["weights"]
    at = torch.arange(w.shape[2], device=w.device)
    held = s["lengths"].long()[:, None, None]
    rank = torch.where(at >= held, -math.inf, torch.where(at >= held - c["recent"], math.inf, w))
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    w[:, :, :keep] = w.gather(2, order)
    full = -(-keep // block) * block
    for name in ("k", "v"):
        codes, scales, tail = s[name + "_codes"], s[name + "_scales"], s[name + "_tail"]
        x = torch.zeros(b, kv, full, d, device=w.device)
        x[:, :, :keep] = codes.gather(2, order[..., None].expand(b, kv, keep, d)).float() * scales.gather(2, order // block)[..., None]
        got, scale = _quantise(x, block)
        codes[:, :, :keep] = got[:, :, :keep]
        scales[:, :, :full // block] = scale
        tail[:, :, :keep % block] = x[:, :, keep - keep % block:keep]


def _plain_logits(s):
    """Repetition penalty on every token seen, frequency and presence penalties on those of the answer, biases, then
    -inf where the grammar forbids; the next token is the lowest index of the largest logit."""
    x, n = s["logits"], s["logits"].shape[1]
    at = torch.arange(s["tokens"].shape[1], device=x.device)
    there = at < s["lengths"][:, None]
    answer = there & (at >= s["prompt_lengths"][:, None])
    tokens = s["tokens"].long()
    seen = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, tokens, there.int())
    made = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, tokens, answer.int())
    r = s["repetition"][:, None]
    y = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    y = y - s["frequency"][:, None] * made
    y = y - s["presence"][:, None] * (made > 0)
    if s["bias_ids"] is not None:
        used = torch.arange(s["bias_ids"].shape[1], device=x.device) < s["bias_counts"][:, None]
        y.scatter_add_(1, s["bias_ids"].long(), torch.where(used, s["bias_values"], 0.0))
    if s["allowed"] is not None:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device=x.device)) & 1
        y = torch.where(bits.reshape(x.shape[0], -1)[:, :n] > 0, y, -math.inf)
    s["out"].copy_(y)
    best = y.amax(1, keepdim=True)
    place = torch.where(y == best, torch.arange(n, device=x.device), n).amin(1)
    return torch.where(best[:, 0] > NEG, place, 0).int()


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["op"] == "logits":
        held, _ = _histories(c)
        cells = c["batch"] * c["vocab"]
        return {"bytes": 8 * cells + 4 * sum(held) + (cells // 8 if c["mask"] else 0) + 8 * c["batch"] * c["biases"],
                "flops": 2 * cells}
    kv, d, block, held = c["kv"], c["dim"], c["block"], _lengths(c)
    if c["op"] == "store":
        total = 0
        for n in held:
            end = n + c["rows"]
            values = 4 * (n % block) + 4 * c["rows"]  # the open block's earlier rows and the new ones
            codes = end - n // block * block
            kept = 4 * min(c["rows"], end % block)  # the new rows that stay in the open block
            total += 2 * kv * (d * (values + codes + kept) + 4 * (-(-end // block) - n // block))
        return {"bytes": total, "flops": total // 2}
    if c["op"] == "attend":
        t, h = c["rows"], c["heads"]
        slots = sum(n + t for n in held)
        pairs = sum(t * n + t * (t + 1) // 2 for n in held)
        return {"bytes": 2 * kv * slots * d + 8 * kv * slots // block + 8 * c["batch"] * t * h * d + (8 * kv * slots if c["weights"] else 0),
                "flops": 4 * pairs * h * d}
    keep = c["keep"]
    return {"bytes": kv * (4 * sum(held) + c["batch"] * (4 * keep + 2 * (2 * keep * d + 8 * keep // block))),
            "flops": 4 * kv * c["batch"] * keep * d}


# ---------------------------------------------------------------- the same in 64 bits, written apart

def exact(case, seed):
    """What `run` returns, in 64 bits.  Codes are whole numbers defined by the 32-bit steps above, so they have no other
    value here."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"store": _exact_store, "attend": _exact_attend, "evict": _exact_evict, "logits": _exact_logits}[case["op"]](s)


def _block_scales(x, block):
    """[kv, n, d] -> [kv, ceil(n / block)] in 64 bits, the last block as long as it is."""
    return torch.stack([p.abs().amax((1, 2)) / 127.0 for p in x.split(block, 1)], 1)


def _exact_store(s):
    c = s["case"]
    block, t = c["block"], c["rows"]
    result = {}
    for name in ("k", "v"):
        scales, tail = s[name + "_scales"].double(), s[name + "_tail"].double()
        new = s[name].reshape(c["batch"], t, c["kv"], c["dim"]).double()
        for b, n in enumerate(_lengths(c)):
            x = torch.cat([tail[b, :, :n % block].clone(), new[b].transpose(0, 1)], 1)
            got = _block_scales(x, block)
            scales[b, :, n // block:n // block + got.shape[1]] = got
            left = (n + t) % block
            tail[b, :, :left] = x[:, x.shape[1] - left:]
        result |= {name + "_codes": None, name + "_scales": scales, name + "_tail": tail}
    return result


def _exact_attend(s):
    c = s["case"]
    block, t, d, kv = c["block"], c["rows"], c["dim"], c["kv"]
    group = c["heads"] // kv
    q = s["q"].reshape(c["batch"], t, kv, group, d)
    out = torch.empty(c["batch"], t, kv, group, d, dtype=torch.float64, device=q.device)
    weights = s["weights"].double() if c["weights"] else None
    for b, n in enumerate(_lengths(c)):
        m = n + t
        for h in range(kv):
            scale = [s[x + "_scales"][b, h].double().repeat_interleave(block)[:m, None] for x in ("k", "v")]
            k, v = (s[x + "_codes"][b, h, :m].double() * y for x, y in zip(("k", "v"), scale))
            z = torch.einsum("tgd,jd->tgj", q[b, :, h].double(), k) / math.sqrt(d)
            late = torch.arange(m, device=q.device) > n + torch.arange(t, device=q.device)[:, None]
            p = torch.softmax(z.masked_fill(late[:, None], -math.inf), -1)
            out[b, :, h] = torch.einsum("tgj,jd->tgd", p, v)
            if weights is not None:
                weights[b, h, :m] += p.sum((0, 1))
    out = out.reshape(c["batch"] * t, c["heads"] * d)
    return {"out": out, "weights": weights} if c["weights"] else {"out": out}


def _exact_evict(s):
    c = s["case"]
    block, keep = c["block"], c["keep"]
    w = s["weights"].double()
    result = {}
    old = {n: (s[n + "_codes"], s[n + "_scales"].double(), s[n + "_scales"].double().clone(), s[n + "_tail"].double()) for n in ("k", "v")}
    for b, n in enumerate(_lengths(c)):
        for h in range(c["kv"]):
            mine = w[b, h, :n - c["recent"]].cpu().numpy()
            heavy = (-mine).argsort(kind="stable")[:keep - c["recent"]]
            kept = torch.tensor(sorted(heavy.tolist()) + list(range(n - c["recent"], n)), device=w.device)
            w[b, h, :keep] = w[b, h][kept]
            for codes, before, after, tail in old.values():
                x = codes[b, h][kept].double() * before[b, h][kept // block, None]
                got = _block_scales(x[None], block)[0]
                after[b, h, :got.shape[0]] = got
                tail[b, h, :keep % block] = x[keep - keep % block:]
    for name, (_, _, after, tail) in old.items():
        result |= {name + "_codes": None, name + "_scales": after, name + "_tail": tail}
    return result | {"weights": w}


def _exact_logits(s):
    y = s["logits"].double()
    n = y.shape[1]
    token = []
    held, prompt = _histories(s["case"])
    for b in range(y.shape[0]):
        line = s["tokens"][b, :held[b]].long()
        past = line.unique()
        z = y[b, past]
        r = float(s["repetition"][b])
        y[b, past] = torch.where(z > 0, z / r, z * r)
        made, often = line[prompt[b]:].unique(return_counts=True)
        y[b, made] -= float(s["frequency"][b]) * often + float(s["presence"][b])
        if s["bias_ids"] is not None:
            e = int(s["bias_counts"][b])
            y[b, s["bias_ids"][b, :e].long()] += s["bias_values"][b, :e].double()
        if s["allowed"] is not None:
            at = torch.arange(n, device=y.device)
            y[b, (s["allowed"][b].long()[at // 32] >> (at % 32)) & 1 == 0] = -math.inf
        token.append(int(y[b].argmax()) if float(y[b].max()) > NEG else 0)
    return {"logits": y, "token": torch.tensor(token, dtype=torch.int32)}
