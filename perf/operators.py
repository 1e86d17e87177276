"""Performance cases of the decoder-attention operators: rotary positions, the paged key/value cache and the attention
that reads it.  Public entry points: llcompiler_b200.executor.rotary, kv_append and paged_attention.

A case's "op" names the operator.  Lengths of a ragged batch follow from the case alone (spread evenly between the
bounds, in a fixed disorder), the values from the seed.  Cache memory is what a serving process has: pages in random
order, leftovers of earlier sequences in every slot that is not written, table entries past a sequence's pages -1.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # an image encoder's first layer: two images of 13 x 17 patches, queries and keys of 12 heads, fp32, axes (h, w)
        _rotary("rotary_image_f32", tokens=442, heads=24, d=64, pairs=32, axes=2, dtype="f32", interleaved=False),
        # a video encoder: 16 frames of 36 x 36 patches, queries and keys of 16 heads, axes (t, h, w)
        _rotary("rotary_video_bf16", tokens=20736, heads=32, d=128, pairs=64, axes=3, dtype="bf16", interleaved=False),
        # one decoding step of 64 sequences: one token each
        _append("append_decode_b64", batch=64, new_min=1, new_max=1, len_min=1, len_max=4096, heads=32, kv_heads=8, d=128,
                pairs=64, axes=1, page=16, dtype="bf16", interleaved=False, heads_first=False),
        # prompts of five sequences with pictures in them (three axes), partly after an earlier part of the prompt
        _append("append_prompt_b5", batch=5, new_min=1111, new_max=5003, len_min=5003, len_max=9001, heads=32, kv_heads=8, d=128,
                pairs=64, axes=3, page=64, dtype="bf16", interleaved=False, heads_first=False),
        # the least: one token after a short prompt, twelve heads of 64
        _attend("decode_b1_short", batch=1, new_min=1, new_max=1, len_min=77, len_max=77, heads=12, kv_heads=12, d=64, page=16,
                window=0, sinks=0, dtype="bf16", heads_first=False),
        # a decoding step of a chat batch
        _attend("decode_b16", batch=16, new_min=1, new_max=1, len_min=100, len_max=4096, heads=32, kv_heads=8, d=128, page=16,
                window=0, sinks=0, dtype="bf16", heads_first=False),
        # a decoding step over long documents, bound by the cache's bytes
        _attend("decode_b32_long", batch=32, new_min=1, new_max=1, len_min=8192, len_max=16384, heads=32, kv_heads=8, d=128, page=64,
                window=0, sinks=0, dtype="bf16", heads_first=False),
        # one very long sequence: the work has to be split over its keys
        _attend("decode_b1_131071", batch=1, new_min=1, new_max=1, len_min=131071, len_max=131071, heads=32, kv_heads=8, d=128, page=128,
                window=0, sinks=0, dtype="bf16", heads_first=True),
        # sliding-window layers of a decoding step: 1024 keys and 4 first ones of up to 32768
        _attend("decode_window_sinks_b48", batch=48, new_min=1, new_max=1, len_min=5000, len_max=32768, heads=64, kv_heads=8, d=64, page=32,
                window=1024, sinks=4, dtype="f16", heads_first=False),
        # chunks of many sizes in one step, single tokens among them; three query heads to a key head
        _attend("chunk_ragged_f16", batch=9, new_min=1, new_max=301, len_min=301, len_max=2048, heads=12, kv_heads=4, d=64, page=16,
                window=0, sinks=0, dtype="f16", heads_first=True),
        # two long prompts in a sliding-window layer
        _attend("chunk_window_4096", batch=2, new_min=4001, new_max=4096, len_min=4500, len_max=6144, heads=16, kv_heads=4, d=128, page=64,
                window=1023, sinks=5, dtype="bf16", heads_first=False),
        # a chunk of 4096 tokens at the end of a prompt of 16384: bound by the tensor cores
        _attend("chunk_4096_of_16384", batch=1, new_min=4096, new_max=4096, len_min=16384, len_max=16384, heads=32, kv_heads=8, d=128, page=64,
                window=0, sinks=0, dtype="bf16", heads_first=False),
    ]


def _rotary(name, **kw):
    return {"name": name, "op": "rotary", **kw}


def _append(name, **kw):
    return {"name": name, "op": "append", **kw}


def _attend(name, **kw):
    return {"name": name, "op": "attend", **kw}


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend"])
    d = rng.choice([64, 128])
    if op == "rotary":
        pairs = rng.choice([d // 2, d // 2, d // 4])
        return {"op": op, "tokens": _log(rng, 1, 20736), "heads": _log(rng, 1, 32), "d": d, "pairs": pairs, "axes": rng.randint(1, 3),
                "dtype": rng.choice(["f32", "bf16", "f16"]), "interleaved": rng.random() < 0.5}
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    c = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "d": d, "page": page, "heads_first": rng.random() < 0.5}
    if op == "append":
        batch = _log(rng, 1, 64)
        new = _log(rng, 1, max(2, 12000 // batch))
        lo = rng.choice([0, 1, new, max(1, new // 2)])
        length = new + _log(rng, 1, max(2, min(8192, 300000 // batch)))
        return {**c, "batch": batch, "new_min": min(lo, new), "new_max": new, "len_min": new, "len_max": length, "pairs": rng.choice([d // 2, d // 4]),
                "axes": rng.randint(1, 3), "dtype": rng.choice(["f32", "bf16", "f16"]), "interleaved": rng.random() < 0.5}
    c["dtype"] = rng.choice(["bf16", "f16"])
    if rng.random() < 0.5:                                   # a decoding step
        batch = _log(rng, 1, 128)
        length = _log(rng, 1, max(2, 400000 // batch))
        new_min = new_max = 1
    else:                                                    # chunks
        batch = _log(rng, 1, 16)
        new_max = _log(rng, 2, 4096)
        new_min = rng.choice([0, 1, new_max, (new_max + 1) // 2])
        room = 1_000_000_000 // (batch * c["heads"] * new_max)   # scores of the padded batch
        length = new_max + _log(rng, 1, max(2, min(room, 200000 // batch)))
        if length * new_max * batch * c["heads"] > 2_000_000_000:
            batch = 1
    windowed = rng.random() < 0.4
    return {**c, "batch": batch, "new_min": new_min, "new_max": new_max, "len_min": max(new_max, length // rng.choice([1, 2, 8])), "len_max": length,
            "window": _log(rng, 1, 4096) if windowed else 0, "sinks": rng.choice([0, 1, 4, 17, 130]) if windowed else 0}


# ---- shapes that follow from a case --------------------------------------------------------------------------------
def _spread(lo, hi, n, step):
    """n whole numbers from lo to hi, evenly spread, in an order that a fixed step gives."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _step(n, near):
    s = near
    while math.gcd(s, n) != 1:
        s += 1
    return s


def _lengths(c):
    """(new tokens, tokens in the cache after them) of each sequence."""
    n = c["batch"]
    new = _spread(c["new_min"], c["new_max"], n, _step(n, 5))
    length = _spread(c["len_min"], c["len_max"], n, _step(n, 7))
    return new, [max(a, b) for a, b in zip(new, length)]


def _sections(pairs, axes):
    """Pairs of each axis: the later axes get equal shares, the first what is left."""
    share = pairs // axes
    return [pairs - share * (axes - 1)] + [share] * (axes - 1)


def _inv_freq(pairs):
    return 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=DEVICE) / pairs)


def _visible(new, length, window, sinks):
    """Pairs (query, key) that see each other in one sequence, and the keys that some query sees."""
    first = length - new
    if new == 0:
        return 0, 0
    if window == 0:
        return sum(range(first + 1, length + 1)), length
    pairs = 0
    for p in range(first, length):
        lo = max(0, p + 1 - window)
        pairs += p + 1 - lo + min(lo, sinks)
    lo = max(0, first + 1 - window)
    return pairs, length - lo + min(lo, sinks)


def work(c):
    e = SIZE[c["dtype"]]
    if c["op"] == "rotary":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["d"] * e + 8 * c["tokens"] * c["axes"], "flops": 6 * n * c["pairs"]}
    new, length = _lengths(c)
    total = sum(new)
    if c["op"] == "append":
        return {"bytes": 2 * total * (c["heads"] + 2 * c["kv_heads"]) * c["d"] * e + 8 * total * c["axes"] + 16 * c["batch"],
                "flops": 6 * total * (c["heads"] + c["kv_heads"]) * c["pairs"]}
    seen = [_visible(a, b, c["window"], c["sinks"]) for a, b in zip(new, length)]
    return {"bytes": 2 * total * c["heads"] * c["d"] * e + 2 * sum(k for _, k in seen) * c["kv_heads"] * c["d"] * e + 16 * c["batch"],
            "flops": 4 * sum(p for p, _ in seen) * c["heads"] * c["d"]}


# ---- what a program has in hand ------------------------------------------------------------------------------------
def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _positions(g, tokens, axes):
    """Positions of patches: the first axis grows along the sequence, the others are places in a picture of 36 columns."""
    t = torch.arange(tokens, device=DEVICE)
    start = int(torch.randint(0, 1 << 17, (1,), generator=g, device=DEVICE))
    rows = [t // 1296 + start if axes > 1 else t + start, (t // 36) % 36, t % 36]
    return torch.stack(rows[:axes]).to(torch.int64).contiguous()


def _cache(g, c, dtype):
    """A pool of pages with leftovers in it, the page table of the batch and its lengths."""
    new, length = _lengths(c)
    page = c["page"]
    need = [-(-n // page) for n in length]
    pages = sum(need) + 3
    shape = (pages, c["kv_heads"], page, c["d"]) if c["heads_first"] else (pages, page, c["kv_heads"], c["d"])
    k, v = torch.empty(shape, device=DEVICE, dtype=dtype), torch.empty(shape, device=DEVICE, dtype=dtype)
    k.normal_(generator=g)
    v.normal_(generator=g)
    if c["heads_first"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((c["batch"], max(1, max(need))), -1, device=DEVICE, dtype=torch.int32)
    ends = torch.tensor([0] + need, device=DEVICE).cumsum(0)
    col = torch.arange(table.shape[1], device=DEVICE)
    held = col[None] < (ends[1:] - ends[:-1])[:, None]
    table[held] = order[: sum(need)]
    q_start = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    kv_len = torch.tensor(length, device=DEVICE, dtype=torch.int32)
    return {"k_cache": k, "v_cache": v, "page_table": table, "q_start": q_start, "kv_len": kv_len, "tokens": sum(new)}


def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, d = DTYPE[c["dtype"]], c["d"]
    s = {"case": c}
    if c["op"] == "rotary":
        # queries and keys are columns of the projection's output [tokens, 3 * heads / 2 * d]
        qkv = _randn(g, (c["tokens"], (c["heads"] + (c["heads"] + 1) // 2) * d), dtype)
        s["x"] = qkv[:, : c["heads"] * d].view(c["tokens"], c["heads"], d)
        s["positions"] = _positions(g, c["tokens"], c["axes"])
    else:
        s.update(_cache(g, c, dtype))
        t, h, hk = s["tokens"], c["heads"], c["kv_heads"]
        if c["op"] == "append":
            qkv = _randn(g, (t, (h + 2 * hk) * d), dtype).view(t, h + 2 * hk, d)
            s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h : h + hk], qkv[:, h + hk :]
            s["positions"] = _positions(g, t, c["axes"])
        else:
            s["q"] = _randn(g, (t, h, d), dtype)
    if "pairs" in c:
        s["inv_freq"], s["sections"] = _inv_freq(c["pairs"]), _sections(c["pairs"], c["axes"])
        s["axis_of_pair"] = torch.repeat_interleave(torch.arange(c["axes"], device=DEVICE), torch.tensor(s["sections"], device=DEVICE), output_size=c["pairs"])
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _turn(x, positions, s):
    """x [tokens, heads, d] turned by its angles, in 32 bits (the angles in 64)."""
    c = s["case"]
    p = c["pairs"]
    angle = positions[s["axis_of_pair"]].t().double() * s["inv_freq"]          # [tokens, pairs]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.float()
    if c["interleaved"]:
        a, b = x[..., 0 : 2 * p : 2], x[..., 1 : 2 * p : 2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p : 2 * p]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., 2 * p :]], -1)


def _plain_append(s):
    c = s["case"]
    t = torch.arange(s["tokens"], device=DEVICE)
    start = s["q_start"].long()
    seq = torch.bucketize(t, start[1:], right=True)
    place = s["kv_len"].long()[seq] - (start[1:] - start[:-1])[seq] + (t - start[seq])
    page, slot = s["page_table"].long()[seq, place // c["page"]], place % c["page"]
    dtype = s["k"].dtype
    s["k_cache"][page, slot] = _turn(s["k"], s["positions"], s).to(dtype)
    s["v_cache"][page, slot] = s["v"]
    return {"q": _turn(s["q"], s["positions"], s).to(dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    c = s["case"]
    h, hk, d, window, sinks = c["heads"], c["kv_heads"], c["d"], c["window"], c["sinks"]
    group = h // hk
    start, length = s["q_start"].long(), s["kv_len"].long()
    new = start[1:] - start[:-1]
    most_new, most_len = c["new_max"], s["page_table"].shape[1] * c["page"]
    b = c["batch"]
    j = torch.arange(most_len, device=DEVICE)
    table = s["page_table"].long().clamp(min=0)
    i = torch.arange(most_new, device=DEVICE)
    at = (start[:-1, None] + i).clamp(max=max(0, s["tokens"] - 1))                   # [b, i]: rows of q
    here = i < new[:, None]
    pos = length[:, None] - new[:, None] + i
    sees = (j <= pos[..., None]) & here[..., None]
    if window:
        sees &= (j > pos[..., None] - window) | (j < sinks)                       # [b, i, j]
    k = s["k_cache"][table].reshape(b, most_len, hk, d).permute(0, 2, 3, 1).float()   # [b, hk, d, j]
    q = s["q"][at].float().reshape(b, most_new, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * most_new, d)
    score = torch.matmul(q, k).view(b, hk, group, most_new, most_len)
    del k
    score *= 1.0 / math.sqrt(d)
    score.masked_fill_(~sees[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top == float("-inf"), torch.zeros_like(top), top)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    v = s["v_cache"][table].reshape(b, most_len, hk, d).permute(0, 2, 1, 3).float()
    v = torch.where((j < length[:, None])[:, None, :, None], v, torch.zeros((), device=DEVICE))
    out = torch.matmul(score.view(b, hk, group * most_new, most_len), v).view(b, hk, group, most_new, d)
    out = torch.where(total > 0, out / total, torch.zeros((), device=DEVICE))
    out = out.permute(0, 3, 1, 2, 4).reshape(b, most_new, h, d)
    return out[here].to(s["q"].dtype)                                          # sequences one after the other


def run(s):
    c = s["case"]
    if own:
        from llcompiler_b200.executor import kv_append, paged_attention, rotary
        if c["op"] == "rotary":
            return rotary(s["x"], s["positions"], s["inv_freq"], sections=s["sections"], interleaved=c["interleaved"])
        if c["op"] == "append":
            q = kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["q_start"], s["kv_len"], q=s["q"], positions=s["positions"],
                          inv_freq=s["inv_freq"], sections=s["sections"], interleaved=c["interleaved"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["q_start"], s["kv_len"], window=c["window"], sinks=c["sinks"],
                               max_q=c["new_max"])
    if c["op"] == "rotary":
        return _turn(s["x"], s["positions"], s).to(s["x"].dtype)
    return _plain_append(s) if c["op"] == "append" else _plain_attend(s)


# ---- in 64 bits ----------------------------------------------------------------------------------------------------
def _exact_turn(x, positions, c):
    """Each pair as a complex number, times e^(i angle)."""
    p, axes = c["pairs"], c["axes"]
    share = p // axes if axes > 1 else 0
    out = x.double().clone()
    for i in range(p):
        axis = 0 if i < p - share * (axes - 1) else 1 + (i - (p - share * (axes - 1))) // share
        angle = positions[axis].double() * 10000.0 ** (-i / p)
        re, im = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + p)
        z = torch.complex(x[..., re].double(), x[..., im].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
        out[..., re], out[..., im] = z.real, z.imag
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rotary":
        return _exact_turn(s["x"], s["positions"], c)
    new, length = _lengths(c)
    table = s["page_table"].tolist()
    if c["op"] == "append":
        q, k = _exact_turn(s["q"], s["positions"], c), _exact_turn(s["k"], s["positions"], c)
        # the caches' other slots hold what they held: as the cache's type in 64 bits
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        row = 0
        for b, (n, full) in enumerate(zip(new, length)):
            place = torch.arange(full - n, full, device=DEVICE)
            page = torch.tensor(table[b], device=DEVICE)[place // c["page"]]
            kc[page, place % c["page"]], vc[page, place % c["page"]] = k[row : row + n], s["v"][row : row + n].double()
            row += n
        return {"q": q, "k_cache": kc, "v_cache": vc}
    h, hk, d = c["heads"], c["kv_heads"], c["d"]
    out = torch.zeros((s["tokens"], h, d), device=DEVICE, dtype=torch.float64)
    row = 0
    for b, (n, full) in enumerate(zip(new, length)):
        if n == 0:
            continue
        first = max(0, full - n + 1 - c["window"]) if c["window"] else 0       # the earliest key inside a window
        keys = torch.cat([torch.arange(min(first, c["sinks"]), device=DEVICE), torch.arange(first, full, device=DEVICE)])
        page = torch.tensor(table[b], device=DEVICE)[keys // c["page"]]
        for g in range(hk):
            kk, vv = s["k_cache"][page, keys % c["page"], g].double(), s["v_cache"][page, keys % c["page"], g].double()
            for x in range(g * (h // hk), (g + 1) * (h // hk)):
                for lo in range(0, n, 2048):
                    hi = min(n, lo + 2048)
                    pos = torch.arange(full - n + lo, full - n + hi, device=DEVICE)[:, None]
                    far = keys[None] > pos
                    if c["window"]:
                        far |= (pos - keys[None] >= c["window"]) & (keys[None] >= c["sinks"])
                    w = (s["q"][row + lo : row + hi, x].double() @ kk.t() / math.sqrt(d)).masked_fill(far, -math.inf)
                    out[row + lo : row + hi, x] = torch.softmax(w, -1) @ vv
        row += n
    return out
