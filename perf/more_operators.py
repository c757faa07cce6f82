"""Measured cases of the 4-bit paged cache and of the head norms: attention of a chunk of new tokens over a cache held
in 4 bits (`Context.op_chunk_attention` on a `PagedKV` of bytes), keys and values quantised as they are written and
read back (`Context.op_kv_append`, `Context.op_kv_read`), reading whole sequences back, and queries and keys
normalised for each head and rotated on their way into the cache (`q_norm`, `k_norm` of `Context.op_kv_append`).

The batch is that of the paged-cache operators: `row_start` [B + 1] cuts the packed rows, `kv_len` [B] counts a
sequence's keys with its chunk, `block_table` [B][max_pages] names its pages of 64 tokens. Token i of a chunk of n is at
position kv_len - n + i. A query at position p sees key j when j < prefix, or j <= p and (no window or j > p - window).

4-bit cache: bytes [page][layer][K, V][kv head][64][9 / 16 head dim]. A block of 64 tokens holds the codes of all
tokens, head dim / 2 bytes each, then their scales, head dim / 32 F16 each: element e of a token has the value
scale[e / 32] * (code[e] - 8). Eight elements 8 w .. 8 w + 7 are a 32-bit word, element e at bits 4 (e % 8); word w
stands at place (w % 4) * (head dim / 32) + w / 4 of its token. A group of 32 with the largest magnitude at m (both
signs have it: the negative one) has the scale -m / 8, kept within +- 2720, rounded to BF16 and then to F16, and the
codes floor(x / scale + 8.5) kept within 0 .. 15, with x / scale as x * (1 / scale) in 32 bits (scale 0: codes 8).

Head norm: y = x * (1 / sqrt(mean(x^2) + eps)) * weight over a head's elements, the sum of the squares rounded once.

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
EPS = 1e-6

# type: of the queries and outputs beside a 4-bit cache, or of the float cache ("append"); rows: of the rows given
ATTENTION = dict(op="attention", type="f16", batch=1, q_min=1, q_max=1, kv_min=1, kv_max=1, heads=16, kv_heads=16,
                 dim=32, layers=2, window=0, prefix=0)
APPEND = dict(op="append", type="f16", rows="f32", batch=1, q_min=1, q_max=1, kv_min=1, kv_max=1, heads=16,
              kv_heads=16, dim=32, layers=2, rot=32, pairs=False, norm=True)
STORE = dict(APPEND, op="store")
READ = dict(op="read", type="f16", rows="f16", batch=1, kv_min=1, kv_max=1, kv_heads=16, dim=32, layers=2)


def listed():
    return [
        # the first decode steps of one request: latency alone counts
        dict(ATTENTION, name="q4_decode_first_steps", kv_min=200, kv_max=200),
        # one decode step of the serving configuration: 64 slots, 16 heads x 32, contexts of a running job
        dict(ATTENTION, name="q4_decode_64_slots", batch=64, kv_min=600, kv_max=2100),
        # decode of a grouped-query backbone, ragged contexts
        dict(ATTENTION, name="q4_decode_grouped", type="bf16", batch=32, kv_min=1000, kv_max=9000, heads=32, kv_heads=8,
             dim=128),
        # one listener on a very long context, what a 4-bit cache is for
        dict(ATTENTION, name="q4_decode_one_long", type="bf16", kv_min=131072, kv_max=131072, heads=32, kv_heads=8,
             dim=128, layers=1),
        # ragged prompt chunks behind cached prefixes, a sliding window over the audio, the text prefix always in view
        dict(ATTENTION, name="q4_chunk_window", batch=3, q_min=333, q_max=1201, kv_min=2500, kv_max=5555, heads=16,
             kv_heads=4, dim=64, window=1024, prefix=150),
        # a prompt's chunk behind the part that is cached already: the largest
        dict(ATTENTION, name="q4_chunk_long", type="bf16", q_min=2048, q_max=2048, kv_min=16384, kv_max=16384, heads=32,
             kv_heads=8, dim=128, layers=1),
        # normalised and rotated, one token for each of 64 slots: latency alone counts
        dict(APPEND, name="norm_append_64_slots", batch=64, kv_min=600, kv_max=2100),
        # the same for prompt chunks of a grouped-query backbone: bandwidth
        dict(APPEND, name="norm_append_prompts", type="bf16", rows="bf16", batch=16, q_min=1400, q_max=2500, kv_min=2500,
             kv_max=4000, heads=32, kv_heads=8, dim=128, rot=128),
        # quantised as they are written and read back, a few drafted tokens, pairs rotated on half of each head
        dict(STORE, name="q4_store_drafts", batch=5, q_min=1, q_max=77, kv_min=700, kv_max=1300, heads=16, kv_heads=4,
             dim=64, rot=32, pairs=True),
        # prompt chunks into the 4-bit cache, and back as rows: bandwidth
        dict(STORE, name="q4_store_prompts", type="bf16", rows="bf16", batch=16, q_min=1400, q_max=2500, kv_min=2500,
             kv_max=4000, heads=32, kv_heads=8, dim=128, rot=128, norm=False),
        # one slot's context read back, to move it elsewhere
        dict(READ, name="q4_read_slot", kv_min=1371, kv_max=1371),
        # the cached prefixes of a grouped-query backbone read back in 32 bits
        dict(READ, name="q4_read_prefixes", type="bf16", rows="f32", batch=16, kv_min=2500, kv_max=8000, kv_heads=8,
             dim=128),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "drafts", "chunk", "chunk", "append", "store", "store", "read"])
    kv_heads, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([32, 64, 128])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 6, 7, 8, 16])
    while kv_heads * group > 48:
        kv_heads //= 2
    same = dict(type=rng.choice(["f16", "bf16"]), kv_heads=kv_heads, dim=dim, layers=rng.choice([1, 2]))
    heads = kv_heads * group
    if kind == "read":
        batch = _spread(rng, 1, 64)
        kv = _spread(rng, 1, max(2, min(40000, int(8e7 / (kv_heads * dim * batch)))))
        return dict(READ, **same, batch=batch, kv_max=kv, kv_min=max(1, int(kv * rng.uniform(0.2, 1.0))),
                    rows=rng.choice([same["type"], "f32"]))
    if kind in ("append", "store"):
        if kind == "append":
            same["type"] = rng.choice(["f16", "bf16", "bf16", "f32"])
        batch = _spread(rng, 1, 128)
        most = min(40000, int(1.6e8 / (kv_heads * (group + 2) * dim)))
        q = _spread(rng, 1, max(1, most // batch))
        kv = q + _spread(rng, 1, 4000)
        return dict(APPEND if kind == "append" else STORE, **same, heads=heads, batch=batch, q_max=q,
                    q_min=max(1, int(q * rng.uniform(0.2, 1.0))), kv_max=kv,
                    kv_min=max(q, int(kv * rng.uniform(0.5, 1.0))), rows=rng.choice(["f32", same["type"]]),
                    rot=rng.choice([0, dim // 2, dim, dim, dim]), pairs=rng.random() < 0.4,
                    norm=kind == "append" or rng.random() < 0.5)
    case = dict(ATTENTION, **same, heads=heads)
    per_key = 2 * kv_heads * dim * 0.5625
    if kind == "decode":
        batch = _spread(rng, 1, 128)
        kv = _spread(rng, 16, min(131072, max(65, int(3e8 / per_key / batch))))
        case.update(batch=batch, kv_max=kv, kv_min=max(1, int(kv * rng.uniform(0.1, 1.0))))
    elif kind == "drafts":
        batch, q = _spread(rng, 1, 64), rng.randint(2, 16)
        kv = _spread(rng, 32, min(32768, int(1.5e8 / per_key / batch)))
        case.update(batch=batch, q_min=q if rng.random() < 0.5 else 1, q_max=q, kv_max=kv,
                    kv_min=max(q, int(kv * rng.uniform(0.1, 1.0))))
    else:
        q = _spread(rng, 17, 2048)
        kv = q + _spread(rng, 1, 12288)
        batch = _spread(rng, 1, 16)
        much = lambda b: 4.0 * b * q * kv * heads * dim > 3e11 or b * q * kv * heads > 1e9  # noqa: E731
        while batch > 1 and much(batch):
            batch -= 1
        while much(batch) and q > 17:
            q, kv = max(17, q * 2 // 3), max(18, kv * 2 // 3)
        case.update(batch=batch, q_max=q, q_min=max(1, int(q * rng.uniform(0.2, 1.0))), kv_max=kv,
                    kv_min=max(q, int(kv * rng.uniform(0.3, 1.0))))
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
        kv.append(int(round(case["kv_min"] + g * (case["kv_max"] - case["kv_min"]))))
        if case["op"] == "read":
            q.append(kv[-1])
            continue
        q.append(int(round(case["q_min"] + f * (case["q_max"] - case["q_min"]))))
        kv[-1] = max(q[-1], kv[-1])
    return q, kv


def _parts(pool, dim):
    """Codes [page][layer][2][kv head][64][dim / 2] and scales [..][64][dim / 16] of a 4-bit pool, as bytes."""
    block = pool.flatten(-2)
    return block[..., :32 * dim].unflatten(-1, (PAGE, dim // 2)), block[..., 32 * dim:].unflatten(-1, (PAGE, dim // 16))


def _quantise(x):
    """Codes [..][dim / 2] and scales [..][dim / 16], as the cache holds them, of f32 values [..][dim]."""
    g = x.unflatten(-1, (-1, 32))
    low, top = g.aminmax(dim=-1)
    scale = (torch.where(-low >= top, low, top) * -0.125).clamp(-2720.0, 2720.0).bfloat16().half()
    wide = scale.float()
    inv = torch.where(wide != 0, 1.0 / wide, 0.0)
    code = (g * inv[..., None] + 8.5).floor().clamp(0.0, 15.0).to(torch.uint8)
    code = code.unflatten(-1, (4, 4, 2))   # [..][group][word][byte][low, high]
    code = (code[..., 0] | code[..., 1] << 4).transpose(-3, -2)
    return code.flatten(-3), scale.contiguous().view(torch.uint8)


def _values(codes, scales):
    """f32 values [..][dim] of codes [..][dim / 2] and scales [..][dim / 16]."""
    groups = codes.shape[-1] // 16
    words = codes.unflatten(-1, (4, groups, 4)).transpose(-3, -2)   # [..][group][word][byte]
    x = torch.stack((words & 15, words >> 4), -1).flatten(-3).float() - 8.0
    return (x * scales.contiguous().view(torch.float16).float()[..., None]).flatten(-2)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op, ty = case["op"], TYPES[case["type"]]
    q_len, kv_len = _lengths(case)
    batch, kv_heads, dim, layers = (case[k] for k in ("batch", "kv_heads", "dim", "layers"))
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
    s = dict(case=case, layer=layers - 1, table=table, row_start=torch.tensor(starts, dtype=torch.int32, device=dev),
             kv_len=torch.tensor(kv_len, dtype=torch.int32, device=dev), max_q=max(q_len), max_kv=max(kv_len))
    if op == "append":
        pool = torch.empty(n_pages, layers, 2, kv_heads, PAGE, dim, dtype=ty, device=dev)
        pool.view(-1).normal_(generator=gen)
    else:
        pool = torch.empty(n_pages, layers, 2, kv_heads, PAGE, 9 * dim // 16, dtype=torch.uint8, device=dev)
        codes, scales = _parts(pool, dim)
        for i in range(0, n_pages, 512):
            x = torch.randn(*codes[i:i + 512].shape[:-1], dim, generator=gen, device=dev)
            codes[i:i + 512], scales[i:i + 512] = _quantise(x)
    s["pool"] = pool
    row_type = TYPES[case["rows"]] if op != "attention" else ty
    if op == "read":
        s["k"] = torch.empty(rows, kv_heads, dim, dtype=row_type, device=dev)
        s["v"] = torch.empty_like(s["k"])
    else:
        # one fused projection's rows, q | k | v, as a layer leaves them
        heads = case["heads"]
        qkv = torch.empty(rows, heads + 2 * kv_heads, dim, dtype=row_type, device=dev)
        qkv.view(-1).normal_(generator=gen)
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        s["out"] = torch.empty(rows, heads, dim, dtype=ty, device=dev)
    if op == "attention":
        s["lse"] = torch.empty(rows, case["heads"], dtype=torch.float32, device=dev)
        s["prefix"] = None
        if case["prefix"]:
            s["prefix"] = torch.tensor([min(case["prefix"] + i % 7, n) for i, n in enumerate(kv_len)],
                                       dtype=torch.int32, device=dev)
    if op in ("append", "store"):
        s["cos"] = s["sin"] = s["q_norm"] = s["k_norm"] = None
        if case["rot"]:
            turn = torch.tensor([10000.0 ** (-2.0 * i / case["rot"]) for i in range(case["rot"] // 2)],
                                dtype=torch.float64, device=dev)
            ang = torch.arange(s["max_kv"], dtype=torch.float64, device=dev)[:, None] * turn
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (1.0 + 0.2 * torch.randn(2, dim, generator=gen, device=dev)).unbind()
    if op == "store":
        s["k_back"] = torch.empty(rows, kv_heads, dim, dtype=ty, device=dev)
        s["v_back"] = torch.empty_like(s["k_back"])
    if own:
        lib = _library()
        s["cache"] = lib.PagedKV(pool) if op == "append" else lib.PagedKV(pool, rows=ty)
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
    op = s["case"]["op"]
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "store": _plain_store, "read": _plain_read}[op](s)
    if op == "attention":
        _ctx().op_chunk_attention(s["cache"], s["chunks"], s["layer"], s["q"], s["out"], prefix=s["prefix"],
                                  window=s["case"]["window"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "read":
        _ctx().op_kv_read(s["cache"], s["chunks"], s["layer"], s["k"], s["v"])
        return {"k": s["k"], "v": s["v"]}
    _ctx().op_kv_append(s["cache"], s["chunks"], s["layer"], s["q"], s["k"], s["v"], s["out"], cos=s["cos"], sin=s["sin"],
                        pairs=s["case"]["pairs"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    if op == "append":
        return {"q": s["out"], "pool": s["pool"]}
    _ctx().op_kv_read(s["cache"], s["chunks"], s["layer"], s["k_back"], s["v_back"])
    return {"q": s["out"], "k": s["k_back"], "v": s["v_back"]}


def _places(s, rows):
    """Sequence, index in the chunk and cache position of every packed row."""
    at = torch.arange(rows, device=s["table"].device)
    seq = (at[:, None] >= s["row_start"][None, 1:]).sum(1)
    i = at - s["row_start"][seq]
    n = s["row_start"][1:] - s["row_start"][:-1]
    return seq, i, s["kv_len"][seq] - n[seq] + i


def _plain_norm(x, weight):
    if weight is None:
        return x
    mean = (x.double().square().sum(-1, keepdim=True).float()) * (1.0 / x.shape[-1])
    return x * (1.0 / (mean + EPS).sqrt()) * weight


def _plain_rotate(x, cos, sin, pairs):
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    if pairs:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_rows(s):
    """Queries and keys of the rows, normalised and rotated, and their sequences and cache positions."""
    seq, _, place = _places(s, s["k"].shape[0])
    q, k = _plain_norm(s["q"].float(), s["q_norm"]), _plain_norm(s["k"].float(), s["k_norm"])
    if s["cos"] is not None:
        q = _plain_rotate(q, s["cos"][place], s["sin"][place], s["case"]["pairs"])
        k = _plain_rotate(k, s["cos"][place], s["sin"][place], s["case"]["pairs"])
    return q, k, seq, place


def _plain_append(s):
    q, k, seq, place = _plain_rows(s)
    pool = s["pool"]
    page = s["table"][seq, place // PAGE].long()
    pool[page, s["layer"], 0, :, place % PAGE] = k.to(pool.dtype)
    pool[page, s["layer"], 1, :, place % PAGE] = s["v"].to(pool.dtype)
    return {"q": q.to(pool.dtype), "pool": pool}


def _plain_store(s):
    q, k, seq, place = _plain_rows(s)
    page = s["table"][seq, place // PAGE].long()
    codes, scales = _parts(s["pool"], s["case"]["dim"])
    codes[page, s["layer"], 0, :, place % PAGE], scales[page, s["layer"], 0, :, place % PAGE] = _quantise(k)
    codes[page, s["layer"], 1, :, place % PAGE], scales[page, s["layer"], 1, :, place % PAGE] = _quantise(s["v"].float())
    back = _plain_read(s)
    return {"q": q.to(s["out"].dtype), "k": back["k"].to(s["out"].dtype), "v": back["v"].to(s["out"].dtype)}


def _plain_read(s):
    seq, _, place = _places(s, s["k"].shape[0])
    page = s["table"][seq, place // PAGE].long()
    codes, scales = _parts(s["pool"], s["case"]["dim"])
    at = lambda which: _values(codes[page, s["layer"], which, :, place % PAGE],  # noqa: E731
                               scales[page, s["layer"], which, :, place % PAGE])
    return {"k": at(0).to(s["k"].dtype), "v": at(1).to(s["k"].dtype)}


def _plain_attention(s):
    case = s["case"]
    seq, i, place = _places(s, s["q"].shape[0])
    batch, heads, kv_heads, dim = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    group, dev = heads // kv_heads, s["q"].device
    # keys and values of every sequence, [batch][kv head][keys][dim], padded to whole pages
    codes, scales = _parts(s["pool"], dim)
    table = s["table"].long()
    kv = _values(codes[table, s["layer"]], scales[table, s["layer"]])
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, batch, kv_heads, -1, dim)
    key = torch.arange(kv.shape[3], device=dev)
    q = torch.zeros(batch, s["max_q"], kv_heads, group, dim, device=dev)
    q[seq, i] = s["q"].float().view(-1, kv_heads, group, dim)
    p = torch.full((batch, s["max_q"]), -1, dtype=torch.long, device=dev)
    p[seq, i] = place
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim), kv[0].transpose(2, 3))
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
    out = torch.matmul(weights.view(batch, kv_heads, -1, weights.shape[-1]), kv[1])
    out = out.view(batch, kv_heads, group, s["max_q"], dim) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, s["max_q"], heads, dim)[seq, i]
    lse = lse.permute(0, 3, 1, 2).reshape(batch, s["max_q"], heads)[seq, i]
    return {"out": out.to(s["out"].dtype), "lse": lse}


def work(case):
    q_len, kv_len = _lengths(case)
    rows, kv_heads, dim = sum(q_len), case["kv_heads"], case["dim"]
    size, held = SIZE[case["type"]], 0.5625   # bytes of a row's element, of a cached one
    if case["op"] == "read":
        return {"bytes": 2 * rows * kv_heads * dim * (held + SIZE[case["rows"]]), "flops": 2.0 * rows * kv_heads * dim}
    heads = case["heads"]
    if case["op"] in ("append", "store"):
        read = rows * (heads + 2 * kv_heads) * dim * SIZE[case["rows"]]
        if case["rot"]:  # the table's rows, cos and sin, each position once
            read += (case["kv_max"] - min(k - q for q, k in zip(q_len, kv_len))) * case["rot"] * 4
        if case["norm"]:
            read += 2 * dim * 4
        turned = rows * (heads + kv_heads)
        flops = 3.0 * turned * case["rot"] + (4.0 * turned * dim if case["norm"] else 0.0)
        if case["op"] == "append":
            return {"bytes": read + rows * (heads + 2 * kv_heads) * dim * size, "flops": flops}
        written = rows * heads * dim * size + 2 * rows * kv_heads * dim * (held + size)
        return {"bytes": read + written, "flops": flops + 8.0 * rows * kv_heads * dim}
    pairs, keys = 0, 0
    for s, (n, total) in enumerate(zip(q_len, kv_len)):
        prefix = min(case["prefix"] + s % 7, total) if case["prefix"] else 0
        first = total - n
        for p in range(first, total):
            low = max(0, p - case["window"] + 1) if case["window"] else 0
            pairs += p + 1 - low + min(prefix, low) + max(0, prefix - (p + 1))
        low = max(0, first - case["window"] + 1) if case["window"] else 0
        keys += total - low + min(prefix, low)
    return {"bytes": 2 * rows * heads * dim * size + rows * heads * 4 + 2 * keys * kv_heads * dim * held,
            "flops": 4.0 * pairs * heads * dim}


def _exact_cached(s, b, n, which, head):
    """The first n keys or values of sequence b in 64 bits: every element looked up by its own bits."""
    dim = s["case"]["dim"]
    e = torch.arange(dim, device=s["table"].device)
    word, group = e // 8, e // 32
    byte = ((word % 4) * (dim // 32) + word // 4) * 4 + e % 8 // 2
    pages = s["table"][b, :-(-n // PAGE)].long()
    block = s["pool"][pages, s["layer"], which, head].flatten(1)
    token = torch.arange(PAGE, device=e.device)[:, None]
    code = block[:, token * (dim // 2) + byte].long() >> (4 * (e % 2)) & 15
    at = 32 * dim + token * (dim // 16) + 2 * group
    bits = block[:, at].long() | block[:, at + 1].long() << 8
    sign, power, part = bits >> 15, bits >> 10 & 31, (bits & 1023).double()
    scale = torch.where(power > 0, (1024.0 + part) * torch.exp2(power.double() - 25.0), part * 2.0 ** -24)
    return ((code - 8).double() * torch.where(sign > 0, -scale, scale)).flatten(0, 1)[:n]


def _exact_turned(s, x, weight):
    """Rows [rows][heads][dim] normalised and rotated in 64 bits, sequence by sequence."""
    case, x = s["case"], x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    if case["rot"]:
        half = case["rot"] // 2
        first = slice(0, 2 * half, 2) if case["pairs"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["pairs"] else slice(half, 2 * half)
        x = x.clone()
        at = 0
        for n, total in zip(*_lengths(case)):
            turn = torch.complex(s["cos"][total - n:total].double(), s["sin"][total - n:total].double())[:, None]
            rows = x[at:at + n]
            z = torch.complex(rows[..., first].contiguous(), rows[..., second].contiguous()) * turn
            rows[..., first], rows[..., second] = z.real, z.imag
            at += n
    return x


def _exact_held(x):
    """What the cache gives back for values [..][dim], from the quantiser's definition in 64 bits."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[-1], 32):
        y = x[..., g:g + 32]
        big = y.abs().amax(-1, keepdim=True)
        m = torch.where((y == -big).any(-1, keepdim=True), -big, big)
        scale = (m / -8.0).clamp(-2720.0, 2720.0).to(torch.bfloat16).to(torch.float16).double()
        code = torch.floor(y / torch.where(scale == 0, 1.0, scale) + 8.5).clamp(0, 15)
        out[..., g:g + 32] = torch.where(scale == 0, 0.0, (code - 8) * scale)
    return out


def exact(case, seed):
    """The outputs of run() from the definition, in 64 bits: sequence by sequence, kv head by kv head."""
    s = prepare(case, seed)
    kv_heads, dim, layer = case["kv_heads"], case["dim"], s["layer"]
    q_len, kv_len = _lengths(case)
    rows, dev = sum(q_len), s["table"].device
    if case["op"] == "read":
        back = [torch.stack([torch.cat([_exact_cached(s, b, n, which, h) for b, n in enumerate(kv_len)])
                             for h in range(kv_heads)], 1) for which in (0, 1)]
        return {"k": back[0], "v": back[1]}
    if case["op"] == "store":
        return {"q": _exact_turned(s, s["q"], s["q_norm"]), "k": _exact_held(_exact_turned(s, s["k"], s["k_norm"])),
                "v": _exact_held(s["v"].double())}
    if case["op"] == "append":
        pool, k = s["pool"].double(), _exact_turned(s, s["k"], s["k_norm"])
        at = 0
        for b, (n, total) in enumerate(zip(q_len, kv_len)):
            place = torch.arange(total - n, total, device=dev)
            page = s["table"][b].long()[place // PAGE]
            pool[page, layer, 0, :, place % PAGE] = k[at:at + n]
            pool[page, layer, 1, :, place % PAGE] = s["v"][at:at + n].double()
            at += n
        return {"q": _exact_turned(s, s["q"], s["q_norm"]), "pool": pool}
    heads = case["heads"]
    group = heads // kv_heads
    out = torch.empty(rows, heads, dim, dtype=torch.float64, device=dev)
    lse = torch.empty(rows, heads, dtype=torch.float64, device=dev)
    at = 0
    for b, (n, total) in enumerate(zip(q_len, kv_len)):
        place = torch.arange(total - n, total, device=dev)[:, None]
        key = torch.arange(total, device=dev)[None]
        hidden = key > place
        if case["window"]:
            hidden |= place - key >= case["window"]
        if case["prefix"]:
            hidden &= key >= int(s["prefix"][b])
        for h in range(kv_heads):
            k, v = _exact_cached(s, b, total, 0, h), _exact_cached(s, b, total, 1, h)
            for g in range(h * group, (h + 1) * group):
                x = s["q"][at:at + n, g].double() @ k.T
                x.div_(math.sqrt(dim)).masked_fill_(hidden, -math.inf)
                lse[at:at + n, g] = torch.logsumexp(x, -1)
                out[at:at + n, g] = torch.softmax(x, -1) @ v
        at += n
    return {"out": out, "lse": lse}
