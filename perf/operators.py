"""Measured cases of the paged-cache operators: appending keys and values to the paged KV cache with the
position rotation applied on the way (`Context.op_kv_append`), and attention of a chunk of new tokens over
the paged cache (`Context.op_chunk_attention`).

Cache layout (the library's): pages [page][layer][K, V][kv head][64 tokens][head dim]. A batch is a ragged
list of sequences: `row_start` [B + 1] cuts the packed rows, `kv_len` [B] counts a sequence's keys with its
chunk, `block_table` [B][max_pages] names its pages. Token i of a chunk of n is at position kv_len - n + i.
A query at position p sees key j when j < prefix, or j <= p and (no window or j > p - window).

With `own` false, run() is the plain form: elementary torch operations in 32 bits, rounded once at the end.
With `own` true it makes the library's calls.
"""
import math
import os
import sys

import torch

own = False

PAGE = 64
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}

# What an attention or append case needs; cases name what differs.
ATTENTION = dict(op="attention", type="f16", batch=1, q_min=1, q_max=1, kv_min=1, kv_max=1, heads=16, kv_heads=16,
                 dim=32, layers=2, window=0, prefix=0)
APPEND = dict(op="append", type="f16", rows="f32", batch=1, q_min=1, q_max=1, kv_min=1, kv_max=1, heads=16,
              kv_heads=16, dim=32, layers=2, rot=32, pairs=False, restart=False)


def listed():
    return [
        # the first decode steps of one request: latency alone counts
        dict(ATTENTION, name="decode_first_steps", kv_min=200, kv_max=200),
        # one decode step of the serving configuration: 64 slots, 16 heads x 32, contexts of a running job
        dict(ATTENTION, name="decode_64_slots", batch=64, kv_min=600, kv_max=2100),
        # decode of a grouped-query backbone, ragged contexts
        dict(ATTENTION, name="decode_grouped", type="bf16", batch=32, kv_min=1000, kv_max=9000, heads=32, kv_heads=8,
             dim=128),
        # one listener on a very long context: the keys have to be split over the whole GPU
        dict(ATTENTION, name="decode_one_long", type="bf16", kv_min=131072, kv_max=131072, heads=32, kv_heads=8,
             dim=128, layers=1),
        # a few drafted tokens per sequence, checked in one pass
        dict(ATTENTION, name="drafts_of_5", batch=16, q_min=5, q_max=5, kv_min=500, kv_max=3000, heads=16, kv_heads=4,
             dim=64),
        # the reference-exact F32 cache: text prefix seen by all, audio tokens causal
        dict(ATTENTION, name="chunk_f32_prefix", type="f32", batch=4, q_min=150, q_max=333, kv_min=400, kv_max=1500,
             prefix=117),
        # ragged prompt chunks of several requests behind cached prefixes
        dict(ATTENTION, name="chunk_ragged", type="bf16", batch=4, q_min=200, q_max=901, kv_min=900, kv_max=4500,
             heads=32, kv_heads=8, dim=128),
        # streaming: a sliding window over the audio, the text prefix always in view
        dict(ATTENTION, name="chunk_window", batch=2, q_min=1500, q_max=1999, kv_min=5000, kv_max=7777, heads=16,
             kv_heads=4, dim=64, window=1024, prefix=150),
        # a long prompt's chunk behind the part that is cached already: the largest
        dict(ATTENTION, name="chunk_long", type="bf16", q_min=4096, q_max=4096, kv_min=16384, kv_max=16384, heads=32,
             kv_heads=8, dim=128, layers=1),
        # one token for each of 64 slots: latency alone counts
        dict(APPEND, name="append_64_slots", batch=64, kv_min=600, kv_max=2100),
        # F32 cache, rotation of adjacent pairs on half of each head, positions that restart after the prefix
        dict(APPEND, name="append_pairs_f32", type="f32", batch=5, q_min=77, q_max=501, kv_min=700, kv_max=1300,
             heads=16, kv_heads=4, dim=64, rot=32, pairs=True, restart=True),
        # prompt chunks of a grouped-query backbone: bandwidth
        dict(APPEND, name="append_prompts", type="bf16", rows="bf16", batch=16, q_min=1400, q_max=2500, kv_min=2500,
             kv_max=4000, heads=32, kv_heads=8, dim=128, rot=128),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "drafts", "chunk", "chunk", "append", "append"])
    kv_type = rng.choice(["f16", "bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 6, 7, 8, 16])
    dim = rng.choice([32, 64, 128])
    while kv_heads * group > 48:
        kv_heads //= 2
    case = dict(ATTENTION if kind != "append" else APPEND, type=kv_type, heads=kv_heads * group, kv_heads=kv_heads,
                dim=dim, layers=rng.choice([1, 2]))
    per_key = 2 * kv_heads * dim * SIZE[kv_type]
    if kind == "decode":
        batch = _spread(rng, 1, 128)
        most = min(131072, max(65, int(1.2e9 / per_key / batch)))
        kv = _spread(rng, 16, most)
        case.update(batch=batch, kv_max=kv, kv_min=max(1, int(kv * rng.uniform(0.1, 1.0))))
    elif kind == "drafts":
        batch, q = _spread(rng, 1, 64), rng.randint(2, 16)
        kv = _spread(rng, 32, min(32768, int(6e8 / per_key / batch)))
        case.update(batch=batch, q_min=q if rng.random() < 0.5 else 1, q_max=q, kv_max=kv,
                    kv_min=max(q, int(kv * rng.uniform(0.1, 1.0))))
    elif kind == "chunk":
        q = _spread(rng, 17, 4096)
        kv = q + _spread(rng, 1, 12288)
        cost = lambda b: 4.0 * b * q * kv * case["heads"] * dim * (6 if kv_type == "f32" else 1)  # noqa: E731
        batch = _spread(rng, 1, 16)
        much = lambda b: cost(b) > 4e11 or b * q * kv * case["heads"] > 1.5e9  # noqa: E731
        while batch > 1 and much(batch):
            batch -= 1
        while much(batch) and q > 17:
            q, kv = max(17, q * 2 // 3), max(18, kv * 2 // 3)
        case.update(batch=batch, q_max=q, q_min=max(1, int(q * rng.uniform(0.2, 1.0))), kv_max=kv,
                    kv_min=max(q, int(kv * rng.uniform(0.3, 1.0))))
    else:
        batch = _spread(rng, 1, 128)
        most = min(40000, int(1.8e8 / (kv_heads * (group + 2) * dim)))
        q = _spread(rng, 1, max(1, most // batch))
        kv = q + _spread(rng, 1, 4000)
        case.update(batch=batch, q_max=q, q_min=max(1, int(q * rng.uniform(0.2, 1.0))), kv_max=kv,
                    kv_min=max(q, int(kv * rng.uniform(0.5, 1.0))), rows=rng.choice(["f32", kv_type]),
                    rot=rng.choice([0, dim // 2, dim, dim, dim]), pairs=rng.random() < 0.4,
                    restart=rng.random() < 0.3)
    if kind != "append":
        if rng.random() < 0.3:
            case["window"] = _spread(rng, 16, 4096)
        if rng.random() < 0.3:
            case["prefix"] = _spread(rng, 8, 600)
    return case


def _lengths(case):
    """Chunk lengths and key counts of the sequences: spread evenly over the case's ranges, the largest first."""
    q, kv = [], []
    for i in range(case["batch"]):
        f = 1.0 - (i * 0.6180339887498949) % 1.0
        g = 1.0 - (i * 0.4142135623730951) % 1.0
        q.append(int(round(case["q_min"] + f * (case["q_max"] - case["q_min"]))))
        kv.append(max(q[-1], int(round(case["kv_min"] + g * (case["kv_max"] - case["kv_min"])))))
    return q, kv


def _frequencies(rot, device):
    """Angles per position of the rot / 2 rotated pairs."""
    return torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=device)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    ty = TYPES[case["type"]]
    q_len, kv_len = _lengths(case)
    batch, heads, kv_heads, dim, layers = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "layers"))
    pages = [-(-n // PAGE) for n in kv_len]
    max_pages = max(pages)
    n_pages = sum(pages) + 3
    order = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(batch, max_pages, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in q_len:
        starts.append(starts[-1] + n)
    rows = starts[-1]
    pool = torch.empty(n_pages, layers, 2, kv_heads, PAGE, dim, dtype=ty, device=dev)
    pool.view(-1).normal_(generator=gen)
    # one fused projection's rows, q | k | v, as a layer leaves them
    row_type = TYPES[case["rows"]] if case["op"] == "append" else ty
    width = heads + 2 * kv_heads
    qkv = torch.empty(rows, width, dim, dtype=row_type, device=dev)
    qkv.view(-1).normal_(generator=gen)
    s = dict(case=case, pool=pool, table=table, layer=layers - 1,
             row_start=torch.tensor(starts, dtype=torch.int32, device=dev),
             kv_len=torch.tensor(kv_len, dtype=torch.int32, device=dev),
             q=qkv[:, :heads], k=qkv[:, heads:heads + kv_heads], v=qkv[:, heads + kv_heads:],
             out=torch.empty(rows, heads, dim, dtype=ty, device=dev), max_q=max(q_len), max_kv=max(kv_len))
    if case["op"] == "attention":
        s["lse"] = torch.empty(rows, heads, dtype=torch.float32, device=dev)
        s["prefix"] = None
        if case["prefix"]:
            s["prefix"] = torch.tensor([min(case["prefix"] + i % 7, n) for i, n in enumerate(kv_len)],
                                       dtype=torch.int32, device=dev)
    else:
        s["cos"] = s["sin"] = s["pos"] = None
        if case["rot"]:
            ang = torch.arange(s["max_kv"], dtype=torch.float64, device=dev)[:, None] * _frequencies(case["rot"], dev)
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
            if case["restart"]:
                s["pos"] = torch.cat([torch.arange(n, dtype=torch.int32, device=dev) for n in q_len])
    if own:
        lib = _library()
        s["cache"] = lib.PagedKV(pool)
        s["chunks"] = lib.ChunkBatch(s["row_start"], s["kv_len"], table, rows, s["max_q"])
    return s


_context = None


def _library():
    here = os.path.join(os.getcwd(), "gsv.cpp_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import gsvcu
    return gsvcu


def _ctx():
    global _context
    if _context is None:
        _context = _library().Context(0)
    return _context


def run(s):
    case = s["case"]
    if own:
        if case["op"] == "append":
            _ctx().op_kv_append(s["cache"], s["chunks"], s["layer"], s["q"], s["k"], s["v"], s["out"], cos=s["cos"],
                                sin=s["sin"], pos=s["pos"], pairs=case["pairs"])
            return {"q": s["out"], "pool": s["pool"]}
        _ctx().op_chunk_attention(s["cache"], s["chunks"], s["layer"], s["q"], s["out"], prefix=s["prefix"],
                                  window=case["window"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    return _plain_append(s) if case["op"] == "append" else _plain_attention(s)


def _places(s):
    """Sequence, index in the chunk and cache position of every packed row."""
    rows = s["q"].shape[0]
    at = torch.arange(rows, device=s["q"].device)
    seq = (at[:, None] >= s["row_start"][None, 1:]).sum(1)
    i = at - s["row_start"][seq]
    n = s["row_start"][1:] - s["row_start"][:-1]
    return seq, i, s["kv_len"][seq] - n[seq] + i


def _plain_rotate(x, cos, sin, pairs):
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    x = x.float()
    if pairs:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_append(s):
    seq, _, place = _places(s)
    q, k = s["q"].float(), s["k"].float()
    if s["cos"] is not None:
        pos = place if s["pos"] is None else s["pos"].long()
        q = _plain_rotate(q, s["cos"][pos], s["sin"][pos], s["case"]["pairs"])
        k = _plain_rotate(k, s["cos"][pos], s["sin"][pos], s["case"]["pairs"])
    pool = s["pool"]
    page = s["table"][seq, place // PAGE].long()
    pool[page, s["layer"], 0, :, place % PAGE] = k.to(pool.dtype)
    pool[page, s["layer"], 1, :, place % PAGE] = s["v"].to(pool.dtype)
    return {"q": q.to(pool.dtype), "pool": pool}


def _plain_attention(s):
    case = s["case"]
    seq, i, place = _places(s)
    batch, heads, kv_heads, dim = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    group, dev = heads // kv_heads, s["q"].device
    # keys and values of every sequence, [batch][kv head][keys][dim], padded to whole pages
    kv = s["pool"][s["table"].long(), s["layer"]].permute(2, 0, 3, 1, 4, 5).reshape(2, batch, kv_heads, -1, dim).float()
    key = torch.arange(kv.shape[3], device=dev)
    held = (key[None] < s["kv_len"][:, None])[:, None, :, None]
    k, v = torch.where(held, kv[0], 0.0), torch.where(held, kv[1], 0.0)
    q = torch.zeros(batch, s["max_q"], kv_heads, group, dim, device=dev)
    q[seq, i] = s["q"].float().view(-1, kv_heads, group, dim)
    p = torch.full((batch, s["max_q"]), -1, dtype=torch.long, device=dev)
    p[seq, i] = place
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim), k.transpose(2, 3))
    scores = scores.view(batch, kv_heads, group, s["max_q"], -1) * (1.0 / math.sqrt(dim))
    seen = key <= p[..., None]
    if case["window"]:
        seen &= key > p[..., None] - case["window"]
    if s["prefix"] is not None:
        seen |= key < s["prefix"][:, None, None]
    seen &= key < s["kv_len"][:, None, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(batch, kv_heads, -1, weights.shape[-1]), v)
    out = out.view(batch, kv_heads, group, s["max_q"], dim) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, s["max_q"], heads, dim)[seq, i]
    lse = lse.permute(0, 3, 1, 2).reshape(batch, s["max_q"], heads)[seq, i]
    return {"out": out.to(s["pool"].dtype), "lse": lse}


def work(case):
    q_len, kv_len = _lengths(case)
    rows, heads, kv_heads, dim = sum(q_len), case["heads"], case["kv_heads"], case["dim"]
    size = SIZE[case["type"]]
    if case["op"] == "append":
        read = rows * (heads + 2 * kv_heads) * dim * SIZE[case["rows"]]
        if case["rot"]:  # the table's rows, cos and sin, each position once
            used = max(q_len) if case["restart"] else case["kv_max"] - min(k - q for q, k in zip(q_len, kv_len))
            read += used * case["rot"] * 4
        return {"bytes": read + rows * (heads + 2 * kv_heads) * dim * size,
                "flops": 3.0 * rows * (heads + kv_heads) * case["rot"]}
    pairs, keys = 0, 0
    for s, (n, total) in enumerate(zip(q_len, kv_len)):
        prefix = min(case["prefix"] + s % 7, total) if case["prefix"] else 0
        first = total - n
        for p in range(first, total):
            low = max(0, p - case["window"] + 1) if case["window"] else 0
            pairs += p + 1 - low + min(prefix, low) + max(0, prefix - (p + 1))
        low = max(0, first - case["window"] + 1) if case["window"] else 0
        keys += total - low + min(prefix, low)
    return {"bytes": 2 * rows * heads * dim * size + rows * heads * 4 + 2 * keys * kv_heads * dim * size,
            "flops": 4.0 * pairs * heads * dim}


def exact(case, seed):
    """The outputs of run() from the definition, in 64 bits: sequence by sequence, kv head by kv head."""
    s = prepare(case, seed)
    heads, kv_heads, dim, layer = case["heads"], case["kv_heads"], case["dim"], s["layer"]
    group = heads // kv_heads
    q_len, kv_len = _lengths(case)
    if case["op"] == "append":
        pool, q_out = s["pool"].double(), s["q"].double()
        at = 0
        for b, (n, total) in enumerate(zip(q_len, kv_len)):
            q, k, v = (s[x][at:at + n].double() for x in "qkv")
            place = torch.arange(total - n, total, device=q.device)
            if case["rot"]:
                half = case["rot"] // 2
                t = torch.arange(n, device=q.device) if case["restart"] else place
                turn = torch.complex(s["cos"][t].double(), s["sin"][t].double())[:, None]
                first = slice(0, 2 * half, 2) if case["pairs"] else slice(0, half)
                second = slice(1, 2 * half, 2) if case["pairs"] else slice(half, 2 * half)
                q, k = q.clone(), k.clone()
                for x in (q, k):
                    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
                    x[..., first], x[..., second] = z.real, z.imag
            q_out[at:at + n] = q
            page = s["table"][b].long()[place // PAGE]
            pool[page, layer, 0, :, place % PAGE] = k
            pool[page, layer, 1, :, place % PAGE] = v
            at += n
        return {"q": q_out, "pool": pool}
    out = torch.empty(sum(q_len), heads, dim, dtype=torch.float64, device=s["q"].device)
    lse = torch.empty(sum(q_len), heads, dtype=torch.float64, device=s["q"].device)
    at = 0
    for b, (n, total) in enumerate(zip(q_len, kv_len)):
        place = torch.arange(total - n, total, device=out.device)[:, None]
        key = torch.arange(total, device=out.device)[None]
        hidden = key > place
        if case["window"]:
            hidden |= place - key >= case["window"]
        if case["prefix"]:
            hidden &= key >= int(s["prefix"][b])
        pages = s["table"][b, :-(-total // PAGE)].long()
        for h in range(kv_heads):
            k = s["pool"][pages, layer, 0, h].reshape(-1, dim)[:total].double()
            v = s["pool"][pages, layer, 1, h].reshape(-1, dim)[:total].double()
            for g in range(h * group, (h + 1) * group):
                x = s["q"][at:at + n, g].double() @ k.T
                x.div_(math.sqrt(dim)).masked_fill_(hidden, -math.inf)
                lse[at:at + n, g] = torch.logsumexp(x, -1)
                out[at:at + n, g] = torch.softmax(x, -1) @ v
        at += n
    return {"out": out, "lse": lse}
