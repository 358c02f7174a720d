"""Serving operators around the TurboQuant paged cache, as they are called and in their plain form.

append   keys and values of new tokens: rotary positions, rotation, quantised store into their slots, with the queries of
         the same tokens rotated on the way; then the same slots read back (the values that the cache now stands for)
gather   cached keys and values of chosen slots as 16-bit or 32-bit tensors (what the next chunk of a prefill attends to)
window   decode attention over the last tokens and a few first ones of each sequence
prefix   decode attention of a batch whose sequences begin with the same pages

``own`` false: elementary torch operations.  ``own`` true: the framework's calls.  A cache is
``uint8[blocks, 16, Hk, slot]`` in one of the framework's eight layouts, and queries of the attention cases are raw
(they are multiplied by the rotation on the way), except for FP8 keys, which are not rotated.
"""

import math
import random  # noqa: F401  (the type of draw's argument)
import sys

import torch

own = False

BLOCK = 16
DIM = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# layout: (key bits, value bits, bytes of a token-head), the slot form (AoS) under the same preset
PRESETS = {"soa": (4, 4, 134), "soa_k8": (8, 4, 196), "soa_k3": (3, 4, 118), "soa_k3v3": (3, 3, 102),
           "aos": (4, 4, 134), "aos_k8": (8, 4, 196), "aos_k3": (3, 4, 118), "aos_k3v3": (3, 3, 102)}


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence: the call whose latency every decode step pays
        {"name": "append_1", "op": "append", "n": 1, "hq": 32, "hk": 8, "layout": "soa", "dtype": "bf16", "rotary": 128,
         "interleaved": False, "max_pos": 8192, "padded": 0},
        # a decode step of a large batch on FP8 keys, GQA of eight, some rows of the batch unused
        {"name": "append_256_k8", "op": "append", "n": 256, "hq": 64, "hk": 8, "layout": "soa_k8", "dtype": "fp16",
         "rotary": 128, "interleaved": False, "max_pos": 16384, "padded": 7},
        # an odd chunk of a prefill with its queries, 3-bit slots, half of each head rotated in adjacent pairs
        {"name": "append_2037_k3v3", "op": "append", "n": 2037, "hq": 32, "hk": 8, "layout": "aos_k3v3", "dtype": "bf16",
         "rotary": 64, "interleaved": True, "max_pos": 16384, "padded": 5},
        # a long prefill stored at once (its queries attend before the cache is read)
        {"name": "append_32768", "op": "append", "n": 32768, "hq": 0, "hk": 8, "layout": "soa", "dtype": "bf16",
         "rotary": 128, "interleaved": False, "max_pos": 32768, "padded": 0},
        # the context of a short second chunk, two heads of a sharded model
        {"name": "gather_917_aos", "op": "gather", "n": 917, "hk": 2, "layout": "aos", "dtype": "fp16"},
        # a whole long context before its last chunk
        {"name": "gather_131072", "op": "gather", "n": 131072, "hk": 8, "layout": "soa", "dtype": "bf16"},
        # one long stream: 4096 tokens of 131072 and the first four
        {"name": "window_1_4096", "op": "window", "batch": 1, "hq": 32, "hk": 8, "layout": "soa", "dtype": "bf16",
         "window": 4096, "first": 4, "min_len": 131072, "max_len": 131072, "sinks": False},
        # the headline batch with a window: lengths below, at and above it
        {"name": "window_64_1024", "op": "window", "batch": 64, "hq": 32, "hk": 8, "layout": "soa", "dtype": "bf16",
         "window": 1024, "first": 4, "min_len": 200, "max_len": 4096, "sinks": False},
        # odd window, sink logits, GQA of eight, 3-bit keys, queries in 32 bits
        {"name": "window_37_777_k3", "op": "window", "batch": 37, "hq": 64, "hk": 8, "layout": "soa_k3", "dtype": "fp32",
         "window": 777, "first": 0, "min_len": 1, "max_len": 2600, "sinks": True},
        # a few samples of one prompt on FP8 keys
        {"name": "prefix_5_2048_k8", "op": "prefix", "batch": 5, "hq": 64, "hk": 8, "layout": "soa_k8", "dtype": "bf16",
         "prefix": 2048, "max_own": 77, "sinks": False},
        # the headline batch behind one system prompt of its context length
        {"name": "prefix_64_4096", "op": "prefix", "batch": 64, "hq": 32, "hk": 8, "layout": "soa", "dtype": "bf16",
         "prefix": 4096, "max_own": 512, "sinks": False},
        # the same batch behind a long document
        {"name": "prefix_64_32768", "op": "prefix", "batch": 64, "hq": 32, "hk": 8, "layout": "soa", "dtype": "bf16",
         "prefix": 32768, "max_own": 512, "sinks": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "gather", "window", "prefix"])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 4, 5, 8])
    layout = rng.choice(sorted(PRESETS))
    if op == "append":
        n = _log_int(rng, 1, 12000)
        return {"op": op, "n": n, "hq": rng.choice([0, hq]) if n > 1024 else hq, "hk": hk, "layout": layout,
                "dtype": rng.choice(["bf16", "fp16"]), "rotary": rng.choice([32, 64, 96, 128]),
                "interleaved": rng.random() < 0.5, "max_pos": rng.choice([16384, 40960]), "padded": rng.randint(0, n // 8)}
    if op == "gather":
        return {"op": op, "n": _log_int(rng, 3, 60000), "hk": hk, "layout": layout, "dtype": rng.choice(["bf16", "fp16"])}
    if op == "window":
        batch = _log_int(rng, 1, 96)
        window = _log_int(rng, 16, min(8192, 200000 // batch))
        most = min(65536, window + _log_int(rng, 16, 262144 // batch))
        return {"op": op, "batch": batch, "hq": hq, "hk": hk, "layout": layout, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "window": window, "first": rng.choice([0, 1, 4, 37]), "min_len": rng.randint(1, most), "max_len": most,
                "sinks": rng.random() < 0.3}
    batch = _log_int(rng, 2, 128)
    return {"op": op, "batch": batch, "hq": hq, "hk": hk, "layout": layout, "dtype": "bf16",
            "prefix": BLOCK * _log_int(rng, 8, min(2048, 131072 // batch)), "max_own": _log_int(rng, 1, min(1024, 32768 // batch)),
            "sinks": rng.random() < 0.3}


# ---- inputs -----------------------------------------------------------------------------------------------------------

_BOOKS = {}


def _codebook(bits):
    """Lloyd-Max centroids of N(0, 1/128), float32 (Newton-free fixed point on the closed-form cell means)."""
    if bits not in _BOOKS:
        n = 1 << bits
        c = [-3.0 + 6.0 * (i + 0.5) / n for i in range(n)]
        pdf = lambda x: math.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)  # noqa: E731
        cdf = lambda x: 0.5 * math.erfc(-x / math.sqrt(2))  # noqa: E731
        for _ in range(400):
            e = [-40.0] + [(c[i] + c[i + 1]) / 2 for i in range(n - 1)] + [40.0]
            c = [(pdf(e[i]) - pdf(e[i + 1])) / (cdf(e[i + 1]) - cdf(e[i])) for i in range(n)]
        _BOOKS[bits] = torch.tensor([x / math.sqrt(DIM) for x in c], dtype=torch.float32)
    return _BOOKS[bits]


def _pack(codes, bits):
    """Codes [..., 128] to little-endian bytes, dim d at bit d * bits."""
    c = codes.to(torch.int32).unflatten(-1, (-1, 2 if bits == 4 else 8))
    if bits == 4:
        return (c[..., 0] | (c[..., 1] << 4)).to(torch.uint8)
    word = (c << (3 * torch.arange(8, device=c.device, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    return torch.stack([word & 255, (word >> 8) & 255, word >> 16], -1).flatten(-2).to(torch.uint8)


def _random_cache(g, blocks, hk, layout):
    """A pool of pages as a model's tokens leave them: Gaussian key coordinates, norms around sqrt(128), values of unit
    spread with a scale and zero of their own."""
    kb, vb, slot = PRESETS[layout]
    dev = g.device
    cache = torch.empty(blocks, BLOCK, hk, slot, dtype=torch.uint8, device=dev)
    sigma = 1 / math.sqrt(DIM)
    for b0 in range(0, blocks, 2048):
        n = min(2048, blocks - b0)
        shape = (n, BLOCK, hk)
        if kb == 8:
            keys = torch.randn(*shape, DIM, generator=g, device=dev).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            c = _codebook(kb).to(dev)
            y = torch.randn(*shape, DIM, generator=g, device=dev) * sigma
            keys = _pack(torch.bucketize(y, (c[:-1] + c[1:]) / 2, out_int32=True), kb)
        values = _pack(torch.randint(0, 1 << vb, (*shape, DIM), generator=g, device=dev, dtype=torch.uint8), vb)
        norm = math.sqrt(DIM) * torch.exp(0.15 * torch.randn(*shape, generator=g, device=dev))
        scale = 3.6 / ((1 << vb) - 1) * torch.exp(0.2 * torch.randn(*shape, generator=g, device=dev))
        zero = -0.5 * ((1 << vb) - 1) * scale + 0.2 * torch.randn(*shape, generator=g, device=dev)
        meta = [m.half() for m in ([norm] if kb != 8 else []) + [scale, zero]]
        if layout.startswith("soa"):
            data = torch.cat([keys, values], -1).reshape(n, -1)
            tail = torch.stack(meta, 1).permute(0, 3, 1, 2).contiguous().view(torch.uint8).reshape(n, -1)  # [n, Hk, field, 16]
            cache[b0:b0 + n] = torch.cat([data, tail], -1).reshape(n, BLOCK, hk, slot)
        else:
            m = [x.unsqueeze(-1).view(torch.uint8) for x in meta]
            cache[b0:b0 + n] = torch.cat([keys] + m[:-2] + [values] + m[-2:], -1)
    return cache


def _tables(g, lens, blocks_extra, shared=0):
    """Block table and pool size of sequences of the given lengths: pages from all over the pool, the first ``shared``
    pages of every row the same ones."""
    dev = g.device
    own_pages = [max(0, -(-n // BLOCK) - shared) for n in lens]
    pool = shared + sum(own_pages) + blocks_extra
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(1, shared + max(own_pages)), dtype=torch.int32, device=dev)
    table[:, :shared] = order[:shared]
    at = shared
    for b, n in enumerate(own_pages):
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    return table, pool


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    pick = random.Random(seed)
    s = dict(case)
    hk, layout, dtype = case["hk"], case["layout"], DTYPES[case["dtype"]]
    kb = PRESETS[layout][0]
    s["centroids"] = _codebook(kb).to(dev) if kb != 8 else None
    s["midpoints"] = (s["centroids"][:-1] + s["centroids"][1:]) * 0.5 if kb != 8 else None
    s["rotation"] = torch.linalg.qr(torch.randn(DIM, DIM, generator=g, device=dev, dtype=torch.float64))[0].float().contiguous() \
        if kb != 8 else None
    if case["op"] in ("append", "gather"):
        n = case["n"]
        blocks = -(-n // BLOCK) + 5
        first = pick.randrange(BLOCK)  # the chunk begins inside a page
        pages = torch.randperm(blocks, generator=g, device=dev)
        t = torch.arange(n, device=dev) + first
        slots = (pages[t // BLOCK] * BLOCK + t % BLOCK).to(torch.int32)
        s["cache"] = _random_cache(g, blocks, hk, layout)
        if case["op"] == "gather":
            s["slots"] = slots
            return s
        if case["padded"]:
            slots[torch.randperm(n, generator=g, device=dev)[:case["padded"]]] = -1
        s["slots"] = slots
        hq, r = case["hq"], case["rotary"]
        # keys, values and queries are slices of one projection's output, as a model has them
        qkv = torch.randn(n, (hq + 2 * hk) * DIM, generator=g, device=dev).to(dtype)
        s["query"] = qkv[:, :hq * DIM].unflatten(-1, (hq, DIM)) if hq else None
        s["key"] = qkv[:, hq * DIM:(hq + hk) * DIM].unflatten(-1, (hk, DIM))
        s["value"] = qkv[:, (hq + hk) * DIM:].unflatten(-1, (hk, DIM))
        s["positions"] = pick.randrange(case["max_pos"] - n + 1) + torch.arange(n, device=dev)
        if n < 512:  # a decode step: each token is at its own sequence's end
            s["positions"] = torch.randint(0, case["max_pos"], (n,), generator=g, device=dev)
        freq = 10000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)
        angle = torch.arange(case["max_pos"], device=dev, dtype=torch.float64)[:, None] * freq
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).float()
        return s
    batch, hq = case["batch"], case["hq"]
    if case["op"] == "window":
        lens = [pick.randint(case["min_len"], case["max_len"]) for _ in range(batch)]
        s["table"], pool = _tables(g, lens, 3)
    else:
        lens = [case["prefix"] + pick.randint(1, case["max_own"]) for _ in range(batch)]
        s["table"], pool = _tables(g, lens, 3, case["prefix"] // BLOCK)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["cache"] = _random_cache(g, pool, hk, layout)
    # heads of different sharpness: scores with a spread of about 0.7 to 2.5
    q = torch.randn(batch, hq, DIM, generator=g, device=dev) * (0.7 + 1.8 * torch.rand(hq, 1, generator=g, device=dev))
    s["query"] = q.to(dtype)
    s["sink_logits"] = torch.randn(hq, generator=g, device=dev) * 2 if case["sinks"] else None
    return s


# ---- the passes -------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "append":
        return _append_plain(s)
    if op == "gather":
        k, v = _read(s["cache"], s["slots"].long(), s["layout"], s["centroids"])
        return {"key": k.to(DTYPES[s["dtype"]]), "value": v.to(DTYPES[s["dtype"]])}
    if op == "window":
        return _window_plain(s)
    return _prefix_plain(s)


def _run_own(s):
    sys.path[:0] = ["turboquant-cuda-decode_b200"] if "turboquant-cuda-decode_b200" not in sys.path else []
    import tqb

    op, layout = s["op"], s["layout"]
    if op == "append":
        q = tqb.rope_append(s["key"], s["value"], s["cache"], s["slots"], s["positions"], s["cos_sin"], s["rotation"],
                            s["midpoints"], s["centroids"], layout=layout, interleaved=s["interleaved"], query=s["query"])
        k, v = tqb.gather_kv(s["cache"], s["slots"], s["centroids"], layout=layout, dtype=DTYPES[s["dtype"]])
        return {"key": k, "value": v} if q is None else {"key": k, "value": v, "query": q}
    if op == "gather":
        k, v = tqb.gather_kv(s["cache"], s["slots"], s["centroids"], layout=layout, dtype=DTYPES[s["dtype"]])
        return {"key": k, "value": v}
    if op == "window":
        return tqb.window_attention(s["query"], s["cache"], s["table"], s["lens"], s["rotation"], s["centroids"],
                                    window=s["window"], first_tokens=s["first"], layout=layout, sinks=s["sink_logits"])
    return tqb.prefix_attention(s["query"], s["cache"], s["table"], s["lens"], s["rotation"], s["centroids"],
                                prefix_len=s["prefix"], layout=layout, sinks=s["sink_logits"])


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _unpack(data, bits):
    if bits == 4:
        return torch.stack([data & 15, data >> 4], -1).flatten(-2).long()
    b = data.int().unflatten(-1, (-1, 3))
    word = b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16)
    return ((word.unsqueeze(-1) >> (3 * torch.arange(8, device=data.device, dtype=torch.int32))) & 7).flatten(-2).long()


def _read(cache, slots, layout, centroids):
    """Keys and values, float32 [..., Hk, 128], that the cache holds in ``slots`` [...]; zeros for negative ones."""
    kb, vb, slot = PRESETS[layout]
    blocks, _, hk, _ = cache.shape
    kn, vn = DIM * kb // 8, DIM * vb // 8
    at = slots.clamp(min=0)
    blk, off = at // BLOCK, at % BLOCK
    if layout.startswith("soa"):
        flat = cache.reshape(blocks, -1)
        edge = BLOCK * hk * (kn + vn)
        data = flat[:, :edge].unflatten(-1, (BLOCK, hk, kn + vn))[blk, off]
        meta = flat[:, edge:].view(torch.float16).unflatten(-1, (hk, -1, BLOCK))[blk, :, :, off].float()
        keys, values, norm, scale, zero = data[..., :kn], data[..., kn:], meta[..., :1], meta[..., -2:-1], meta[..., -1:]
    else:
        row = cache[blk, off]
        keys, values = row[..., :kn], row[..., slot - 4 - vn:slot - 4]
        half = lambda i: row[..., i:i + 2].contiguous().view(torch.float16).float()  # noqa: E731
        norm, scale, zero = half(kn), half(slot - 4), half(slot - 2)
    if kb == 8:
        k = keys.contiguous().view(torch.float8_e4m3fn).float()
    else:
        k = centroids[_unpack(keys, kb)]
        if not layout.startswith("soa"):
            k = k / (k.square().sum(-1, keepdim=True) + 1e-16).sqrt()
        k = k * norm
    v = _unpack(values, vb).float() * scale + zero
    live = (slots >= 0)[..., None, None]
    return torch.where(live, k, 0.0), torch.where(live, v, 0.0)


def _rope(x, cs, interleaved):
    """Rotates the first dims of x [N, H, 128] by the cosines and sines cs [N, r] (float64)."""
    x, (c, s) = x.double(), cs.double().unsqueeze(1).chunk(2, -1)
    r = cs.shape[-1]
    turn, rest = x[..., :r], x[..., r:]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)
    a, b = turn.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1)


def _append_plain(s):
    # in 64 bits up to the codes: a coordinate next to a border of the codebook, or a norm next to one of its 16-bit
    # roundings, falls on the other side of it in 32
    kb, vb, _ = PRESETS[s["layout"]]
    dtype = DTYPES[s["dtype"]]
    cs = s["cos_sin"][s["positions"]]
    x = _rope(s["key"], cs, s["interleaved"])
    if kb == 8:
        k = x.float().clamp(-448, 448).to(torch.float8_e4m3fn).float()
    else:
        norm = x.square().sum(-1, keepdim=True).sqrt()
        y = x / (norm + 1e-8) @ s["rotation"].double()
        c = s["centroids"][torch.bucketize(y, s["midpoints"].double(), right=True)]
        size = (c.double().square().sum(-1, keepdim=True) + 1e-16).sqrt()
        if s["layout"].startswith("soa"):  # the stored norm has the length of the centroids folded in
            k = c * (norm / size).half().float()
        else:
            k = c / size.float() * norm.half().float()
    v = s["value"].float()
    low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    top = (1 << vb) - 1
    # a division, not a product with the reciprocal, which a plain number would turn it into
    scale = ((high - low) / torch.full_like(high, top)).clamp(min=1e-8)
    codes = ((v - low) / scale + 0.5).trunc().clamp(0, top)
    v = codes * scale.half().float() + low.half().float()
    live = (s["slots"] >= 0)[:, None, None]
    out = {"key": torch.where(live, k, 0.0).to(dtype), "value": torch.where(live, v, 0.0).to(dtype)}
    if s["query"] is not None:
        q = _rope(s["query"], cs, s["interleaved"])
        out["query"] = (q if kb == 8 else q @ s["rotation"].double()).float()
    return out


def _queries(s):
    q = s["query"].float()
    q = q if s["rotation"] is None else q @ s["rotation"]
    return q.unflatten(1, (s["hk"], -1)) / math.sqrt(DIM)  # [B, Hk, G, 128]


def _slots_of(table, pos):
    return table.gather(1, pos // BLOCK).long() * BLOCK + pos % BLOCK


def _finish(s, w, top, out):
    """Divides the weighted sum by the weights' sum, with the sink logits as one more weight."""
    total = w.sum(-1, keepdim=True)
    if s["sink_logits"] is not None:
        total = total + (s["sink_logits"].unflatten(0, (s["hk"], -1))[None, :, :, None] - top).exp()
    return (out / total).flatten(1, 2).to(DTYPES[s["dtype"]])


def _top(s, score):
    top = score.amax(-1, keepdim=True)
    if s["sink_logits"] is not None:
        top = torch.maximum(top, s["sink_logits"].unflatten(0, (s["hk"], -1))[None, :, :, None])
    return top


def _window_plain(s):
    lens, dev = s["lens"].long()[:, None], s["lens"].device
    low = (lens - s["window"]).clamp(min=0)
    first = torch.arange(s["first"], device=dev)[None]
    pos = torch.cat([first.expand(len(lens), -1), low + torch.arange(s["window"], device=dev)[None]], 1)
    seen = torch.cat([first < low, pos[:, s["first"]:] < lens], 1)
    pos = torch.where(seen, pos, 0)
    k, v = _read(s["cache"], _slots_of(s["table"].long(), pos), s["layout"], s["centroids"])  # [B, T, Hk, 128]
    score = _queries(s) @ k.permute(0, 2, 3, 1)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = _top(s, score)
    w = (score - top).exp()
    return _finish(s, w, top, w @ v.transpose(1, 2))


def _prefix_plain(s):
    lens, dev, p = s["lens"].long()[:, None], s["lens"].device, s["prefix"]
    shared = torch.arange(p, device=dev)[None]
    table = s["table"].long()
    k0, v0 = _read(s["cache"], _slots_of(table[:1], shared)[0], s["layout"], s["centroids"])  # [P, Hk, 128]
    pos = p + torch.arange(s["max_own"], device=dev)[None].expand(len(lens), -1)
    seen = pos < lens
    k1, v1 = _read(s["cache"], _slots_of(table, torch.where(seen, pos, 0)), s["layout"], s["centroids"])
    q = _queries(s)  # [B, Hk, G, 128]
    batch, hk, g, _ = q.shape
    rows = q.transpose(0, 1).reshape(hk, batch * g, DIM)
    one = (rows @ k0.permute(1, 2, 0)).unflatten(1, (batch, g)).transpose(0, 1)  # [B, Hk, G, P]
    two = (q @ k1.permute(0, 2, 3, 1)).masked_fill(~seen[:, None, None], -math.inf)
    score = torch.cat([one, two], -1)
    top = _top(s, score)
    w = (score - top).exp()
    w0 = w[..., :p].transpose(0, 1).reshape(hk, batch * g, p)
    out = (w0 @ v0.transpose(0, 1)).unflatten(1, (batch, g)).transpose(0, 1) + w[..., p:] @ v1.transpose(1, 2)
    return _finish(s, w, top, out)


# ---- the work of a pass -----------------------------------------------------------------------------------------------

def work(case):
    kb, _, slot = PRESETS[case["layout"]]
    hk, size = case["hk"], 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "append":
        n, hq = case["n"], case["hq"]
        moved = n * (hq + 2 * hk) * DIM * size + n * hq * DIM * 4 + 2 * n * hk * slot + 2 * n * hk * DIM * size
        return {"bytes": moved + n * (12 + 4 * case["rotary"]), "flops": 0 if kb == 8 else 2 * DIM * DIM * n * (hq + hk)}
    if case["op"] == "gather":
        return {"bytes": case["n"] * (4 + hk * (slot + 2 * DIM * size)), "flops": 4 * case["n"] * hk * DIM}
    rows = case["batch"] * case["hq"] * DIM * size * 2  # queries in, outputs out
    if case["op"] == "window":
        mean = 0
        for i in range(33):  # lengths are uniform between the two
            n = case["min_len"] + (case["max_len"] - case["min_len"]) * i // 32
            low = max(0, n - case["window"])
            mean += (n - low + min(case["first"], low)) / 33
        tokens = case["batch"] * mean
        return {"bytes": int(rows + tokens * hk * slot), "flops": int(4 * DIM * case["hq"] * tokens)}
    own_tokens = case["batch"] * (1 + case["max_own"]) / 2
    return {"bytes": int(rows + (case["prefix"] + own_tokens) * hk * slot),
            "flops": int(4 * DIM * case["hq"] * (case["batch"] * case["prefix"] + own_tokens))}


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------------

def _field(row, start, bits):
    """128 codes of ``bits`` bits from byte ``start`` on, one dim after another."""
    d = torch.arange(DIM, device=row.device) * bits
    byte = start + d // 8
    two = row[..., byte].long() | (row[..., (byte + 1).clamp(max=row.shape[-1] - 1)].long() << 8)
    return (two >> (d % 8)) & ((1 << bits) - 1)


def _exact_rows(s, slots):
    """The definition of a slot's key and value, float64 [n, Hk, 128], a head at a time."""
    kb, vb, slot = PRESETS[s["layout"]]
    cache, hk = s["cache"], s["hk"]
    raw = cache.reshape(cache.shape[0], -1)[slots // BLOCK]
    t = slots % BLOCK
    kn, vn = DIM * kb // 8, DIM * vb // 8
    fields = 2 if kb == 8 else 3
    pull = lambda start, count: raw.gather(1, start[:, None] + torch.arange(count, device=raw.device))  # noqa: E731
    number = lambda start: pull(start, 2).contiguous().view(torch.float16).double()  # noqa: E731
    keys, values = [], []
    for h in range(hk):
        if s["layout"].startswith("soa"):
            start = (t * hk + h) * (kn + vn)
            meta = BLOCK * hk * (kn + vn) + 2 * (h * fields * BLOCK + t)
            row = pull(start, kn + vn)
            code_at, put = kn, [meta + 2 * BLOCK * i for i in range(fields)]
        else:
            start = (t * hk + h) * slot
            row = pull(start, slot)
            code_at = kn + (0 if kb == 8 else 2)
            put = ([] if kb == 8 else [start + kn]) + [start + slot - 4, start + slot - 2]
        if kb == 8:
            k = row[:, :kn].contiguous().view(torch.float8_e4m3fn).double()
        else:
            k = s["centroids"].double()[_field(row, 0, kb)]
            if s["layout"].startswith("aos"):
                k = k / torch.linalg.vector_norm(k, dim=-1, keepdim=True)
            k = k * number(put[0])
        keys.append(k)
        values.append(_field(row, code_at, vb).double() * number(put[-2]) + number(put[-1]))
    return torch.stack(keys, 1), torch.stack(values, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "gather":
        k, v = _exact_rows(s, s["slots"].long())
        return {"key": k, "value": v}
    return _exact_attention(s)


def _exact_append(s):
    kb, vb, _ = PRESETS[s["layout"]]
    r, n = s["rotary"], s["n"]
    angles = s["cos_sin"].double()[s["positions"]]
    pair = torch.arange(r // 2, device=angles.device)
    i, j = (2 * pair, 2 * pair + 1) if s["interleaved"] else (pair, pair + r // 2)

    def turned(x):
        z = x.double().clone()
        w = torch.complex(x.double()[..., i], x.double()[..., j]) * torch.complex(angles[:, :r // 2], angles[:, r // 2:])[:, None]
        z[..., i], z[..., j] = w.real, w.imag
        return z

    x = turned(s["key"])
    if kb == 8:
        k = x.clamp(-448, 448).to(torch.float8_e4m3fn).double()
    else:
        size = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
        y = torch.einsum("nhd,de->nhe", x, s["rotation"].double()) / (size + 1e-8)
        code = torch.zeros_like(y, dtype=torch.long)
        for m in s["midpoints"].tolist():
            code += y >= m
        c = s["centroids"].double()[code]
        length = torch.linalg.vector_norm(c, dim=-1, keepdim=True)
        k = c * (size / length).half().double() if s["layout"].startswith("soa") else c / length * size.half().double()
    # the grid of a token's values is defined by 32-bit steps (the store's and the reference's): each one is taken in 64
    # bits and rounded to 32, without which a value halfway between two codes has no code of its own
    step32 = lambda x: x.float().double()  # noqa: E731
    v, top = s["value"].double(), (1 << vb) - 1
    low = v.min(-1, keepdim=True).values
    step = step32(step32(v.max(-1, keepdim=True).values - low) / top).clamp(min=step32(torch.tensor(1e-8)).item())
    code = torch.floor(step32(step32(step32(v - low) / step) + 0.5)).clamp(0, top)
    v = code * step.half().double() + low.half().double()
    dead = s["slots"] < 0
    k[dead], v[dead] = 0, 0
    out = {"key": k, "value": v}
    if s["query"] is not None:
        q = turned(s["query"])
        out["query"] = q if kb == 8 else torch.einsum("nhd,de->nhe", q, s["rotation"].double())
    return out


def _exact_attention(s):
    q = s["query"].double()
    q = q if s["rotation"] is None else torch.einsum("bhd,de->bhe", q, s["rotation"].double())
    hk, g = s["hk"], s["hq"] // s["hk"]
    rows, shared = [], None
    if s["op"] == "prefix":
        t = torch.arange(s["prefix"], device=q.device)
        shared = _exact_rows(s, s["table"][0].long()[t // BLOCK] * BLOCK + t % BLOCK)
    for b, n in enumerate(s["lens"].tolist()):
        t = torch.arange(n, device=q.device)
        t = t[t >= s["prefix"]] if s["op"] == "prefix" else t[(t < s["first"]) | (t >= n - s["window"])]
        k, v = _exact_rows(s, s["table"][b].long()[t // BLOCK] * BLOCK + t % BLOCK)
        if shared is not None:
            k, v = torch.cat([shared[0], k]), torch.cat([shared[1], v])
        score = torch.einsum("hgd,thd->hgt", q[b].reshape(hk, g, DIM), k) / math.sqrt(DIM)
        if s["sink_logits"] is not None:  # a key of its own logit and a value of zero
            score = torch.cat([score, s["sink_logits"].double().reshape(hk, g, 1)], -1)
            v = torch.cat([v, torch.zeros_like(v[:1])])
        rows.append(torch.einsum("hgt,thd->hgd", torch.softmax(score, -1), v).reshape(hk * g, DIM))
    return torch.stack(rows)
