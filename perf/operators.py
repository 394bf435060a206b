"""Cases of the attention operators and of the paged key/value cache: sizes, inputs, plain forms, calls, definitions.

Three operators that a model runs one after the other:
  append  qkv_norm_rope_append: per-head norm and rotation of a step's q and k, k and v stored into the cache's pages
  window  attn_window: attention of a packed batch of sequences, with a sliding window and first tokens that stay visible
  decode  attn_decode_paged: attention of one new token of each sequence over the paged cache
"""
import math
import random

import torch

own = False

NONE, INTERLEAVED, HALF = 0, 1, 2
E4M3_MAX = 448.0


# ---- cases ------------------------------------------------------------------------------------------------------

def _append(name, rows, H, Hkv, D, kv, page, **more):
    return dict({"name": name, "op": "append", "rows": rows, "H": H, "Hkv": Hkv, "D": D, "kv": kv, "page": page, "rot": D, "mode": HALF,
                 "packed": True, "k_out": False, "step": False, "idle": 0, "seqs": 1}, **more)


def _window(name, rows, keys, seqs, H, Hkv, D, left, right, sinks, **more):
    return dict({"name": name, "op": "window", "rows": rows, "keys": keys, "seqs": seqs, "H": H, "Hkv": Hkv, "D": D, "left": left,
                 "right": right, "sinks": sinks, "ragged": 0, "packed": False, "behind": 0}, **more)


def _decode(name, seqs, longest, H, Hkv, D, kv, page, **more):
    return dict({"name": name, "op": "decode", "seqs": seqs, "longest": longest, "H": H, "Hkv": Hkv, "D": D, "kv": kv, "page": page,
                 "left": -1, "sinks": 0, "ragged": 0, "heads_first": False}, **more)


def listed():
    return [
        # one token of one sequence: the smallest call there is, all latency
        _append("append-one", 1, 32, 8, 128, "bf16", 16, step=True),
        # a decode step of a served batch, a few of its slots idle, 8-bit cache
        _append("append-step", 250, 32, 8, 128, "e4m3", 64, step=True, idle=6, seqs=256),
        # the prompt's rows of an image batch, rotated in adjacent pairs, with the contiguous keys that attn_window reads
        _append("append-image", 8704, 24, 24, 128, "bf16", 64, mode=INTERLEAVED, packed=False, k_out=True, seqs=2),
        # a video's rows from the packed projection, 96 of 128 channels rotated
        _append("append-video", 33272, 40, 40, 128, "bf16", 128, rot=96, k_out=True),
        # a short prompt of the text encoder: causal, grouped heads, less than one tile of rows
        _window("window-prompt", 77, 77, 1, 32, 8, 128, -1, 0, 0),
        # packed prompts of very different lengths, causal with a window and first tokens, rows behind the last sequence
        _window("window-ragged", 8100, 8100, 9, 32, 8, 128, 1024, 0, 4, ragged=7, behind=92),
        # two images of a batch, everything visible
        _window("window-image", 8704, 8704, 2, 24, 24, 128, -1, -1, 0),
        # one GPU's heads of a video sharded by heads over eight: a window of four frames each way, the first frame stays visible
        _window("window-video", 33272, 33272, 1, 5, 5, 128, 6240, 6240, 1560),
        # one sequence, a short cache: latency
        _decode("decode-short", 1, 500, 32, 8, 128, "bf16", 16),
        # a served batch of uneven lengths, 8-bit cache, narrow heads
        _decode("decode-batch", 48, 9000, 28, 4, 64, "e4m3", 64, ragged=3),
        # a large batch of long sequences
        _decode("decode-long", 64, 16384, 32, 8, 128, "bf16", 16, ragged=5),
        # one very long sequence of grouped heads with a window and first tokens, pages with the head outermost
        _decode("decode-window", 8, 100000, 40, 8, 128, "e4m3", 128, left=32768, sinks=64, heads_first=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "window", "window", "decode", "decode"])
    kv = rng.choice(["bf16", "e4m3"])
    page = rng.choice([16, 16, 24, 32, 64, 100, 128, 256])
    Hkv = rng.choice([1, 2, 4, 5, 8])
    H = Hkv * rng.choice([1, 1, 3, 4, 5, 7, 8])
    D = rng.choice([64, 80, 96, 128, 128, 128])
    if op == "append":
        step = rng.random() < 0.5
        rows = _log(rng, 1, 500) if step else _log(rng, 40, 30000)
        mode = rng.choice([INTERLEAVED, HALF])
        idle = rng.choice([0, 0, rows // 5]) if step else 0
        seqs = rows + idle if step else min(rows, rng.choice([1, 1, 2, 7]))
        return _append("", rows, H, Hkv, D, kv, page, step=step, seqs=seqs, idle=idle, mode=mode, packed=rng.random() < 0.5,
                       rot=rng.choice([D, D, D // 2]), k_out=not step and rng.random() < 0.5)
    if op == "window":
        rows = _log(rng, 1, 9000)
        H = min(H, 40)
        seqs = min(rows, rng.choice([1, 1, 2, 5, 13]))
        keys = rows if rng.random() < 0.6 else rows + seqs * rng.randrange(1, 1000)
        D = rng.choice([64, 72, 80, 128, 128])
        left, right = rng.choice([(-1, -1), (-1, 0), (-1, 0), (_log(rng, 1, 4000), 0), (_log(rng, 16, 2000), _log(rng, 16, 2000))])
        return _window("", rows, keys, seqs, H, Hkv, D, left, right, rng.choice([0, 1, 4, 100]) if left >= 0 else 0,
                       ragged=rng.randrange(1, 1000) if seqs > 1 else 0, packed=keys == rows and rng.random() < 0.3,
                       behind=rng.choice([0, 0, 37]))
    seqs = _log(rng, 1, 200)
    longest = _log(rng, 1, max(8, min(60000, 1100000 // seqs)))
    left, sinks = rng.choice([(-1, 0), (-1, 0), (_log(rng, 1, 4000), rng.choice([0, 4, 64]))])
    return _decode("", seqs, longest, H, Hkv, D, kv, page, left=left, sinks=sinks, ragged=rng.choice([0, rng.randrange(1, 1000)]),
                   heads_first=rng.random() < 0.3)


def _split(total, parts, ragged, least):
    """`parts` lengths that sum to `total`: even ones, or very uneven ones where `ragged` seeds them."""
    if parts == 1:
        return [total]
    if not ragged:
        return [total * (i + 1) // parts - total * i // parts for i in range(parts)]
    rng = random.Random(ragged)
    share = [rng.random() ** 3 + 1e-3 for _ in range(parts)]
    room = total - least * parts
    ends = [0] + [int(room * sum(share[:i + 1]) / sum(share)) for i in range(parts - 1)] + [room]
    return [least + b - a for a, b in zip(ends, ends[1:])]


def _window_lengths(c):
    """(rows, keys) of each sequence; every sequence has the same number of keys more than rows."""
    rows = _split(c["rows"], c["seqs"], c["ragged"], 1)
    return rows, [n + (c["keys"] - c["rows"]) // c["seqs"] for n in rows]


def _decode_lengths(c):
    if not c["ragged"]:
        return [c["longest"]] * c["seqs"]
    rng = random.Random(c["ragged"])
    return [c["longest"]] + [rng.randint(max(1, c["longest"] // 4), c["longest"]) for _ in range(c["seqs"] - 1)]


def _visible(L, p, left, right, sinks):
    """How many of L keys a query at position p sees."""
    hi = L - 1 if right < 0 else min(L - 1, p + right)
    if hi < 0:
        return 0
    if left < 0:
        return hi + 1
    lo = max(0, p - left)
    return max(0, hi + 1 - lo) + min(sinks, lo, hi + 1)


def work(c):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if c["op"] == "append":
        n = c["rows"]
        kv = 2 if c["kv"] == "bf16" else 1
        return {"bytes": n * D * (4 * H + (4 + 2 * kv) * Hkv + (2 * Hkv if c["k_out"] else 0)) + 4 * n * c["rot"],
                "flops": n * D * 8 * (H + Hkv)}
    if c["op"] == "window":
        pairs = 0
        for nq, nk in zip(*_window_lengths(c)):
            pairs += sum(_visible(nk, i + nk - nq, c["left"], c["right"], c["sinks"]) for i in range(nq))
        return {"bytes": 4 * c["rows"] * H * D + 4 * c["keys"] * Hkv * D + 4 * c["rows"] * H, "flops": 4 * D * H * pairs}
    tokens = sum(_visible(n, n - 1, c["left"], 0, c["sinks"]) for n in _decode_lengths(c))
    size = 2 if c["kv"] == "bf16" else 1
    return {"bytes": 2 * tokens * Hkv * D * size + 4 * c["seqs"] * H * D + 4 * c["seqs"] * H, "flops": 4 * tokens * H * D}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _cache(c, g, seqs, longest, fill):
    """Pages in no order, with some to spare; the values of a cache in use, or zeros."""
    page, Hkv, D = c["page"], c["Hkv"], c["D"]
    per = -(-longest // page)
    pages = seqs * per + 3
    shape = (pages, Hkv, page, D) if c.get("heads_first") else (pages, page, Hkv, D)
    kind = torch.bfloat16 if c["kv"] == "bf16" else torch.float8_e4m3fn
    kv, scales = [], []
    for std in (1.3, 1.0):
        scale = None if c["kv"] == "bf16" else (0.02 + 0.02 * torch.rand(Hkv, device="cuda", generator=g)) if c["op"] == "append" else \
            (0.005 + 0.01 * torch.rand(Hkv, device="cuda", generator=g))
        if fill:
            t = torch.randn(shape, device="cuda", generator=g, dtype=torch.bfloat16) * std
            t = t if scale is None else (t * 80).clamp_(-E4M3_MAX, E4M3_MAX).to(kind)  # 80 steps of the scale to the unit
        else:
            t = torch.zeros(shape, device="cuda", dtype=kind if scale is None else torch.uint8).view(kind)
        kv.append(t.transpose(1, 2) if c.get("heads_first") else t)
        scales.append(scale)
    table = torch.randperm(pages, device="cuda", generator=g)[:seqs * per].view(seqs, per).to(torch.int32)
    return kv[0], kv[1], table, scales[0], scales[1]


def _handle(parts):
    if not own:
        return parts
    import miroxen_b200 as mx
    return mx.KvCache(*parts)


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    H, Hkv, D = c["H"], c["Hkv"], c["D"]

    def rand(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.bfloat16) * std

    if c["op"] == "append":
        n, half = c["rows"], c["rot"] // 2
        if c["step"]:  # row t is the next token of a sequence, idle slots among them
            per = 4 * c["page"] + 5
            total = n + c["idle"]
            ids = torch.arange(total, device="cuda", dtype=torch.int32)
            ids[torch.randperm(total, device="cuda", generator=g)[:c["idle"]]] = -1
            pos = torch.randint(0, per, (total,), device="cuda", generator=g, dtype=torch.int32)
        else:
            lens = _split(n, c["seqs"], 0, 1)
            at = [(37 * i + 11) % (2 * c["page"]) for i in range(c["seqs"])]  # tokens that are there already
            per, total = max(a + m for a, m in zip(at, lens)), n
            ids = torch.repeat_interleave(torch.arange(c["seqs"], dtype=torch.int32), torch.tensor(lens)).cuda()
            pos = torch.cat([torch.arange(a, a + m, dtype=torch.int32) for a, m in zip(at, lens)]).cuda()
        if c["packed"]:
            buf = rand(total, (H + 2 * Hkv) * D)
            q, k, v = buf[:, :H * D], buf[:, H * D:(H + Hkv) * D], buf[:, (H + Hkv) * D:]
        else:
            q, k, v = rand(total, H * D), rand(total, Hkv * D), rand(total, Hkv * D)
        angle = torch.arange(per, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        return {"case": c, "q": q, "k": k, "v": v, "ids": ids, "pos": pos,
                "cos": angle.cos().float().cuda(), "sin": angle.sin().float().cuda(),
                "wq": 1 + 0.05 * torch.randn(D, device="cuda", generator=g), "wk": 1 + 0.05 * torch.randn(D, device="cuda", generator=g),
                "cache": _handle(_cache(c, g, c["seqs"], per, False)),
                "q_out": torch.zeros(total, H, D, device="cuda", dtype=torch.bfloat16),
                "k_out": torch.zeros(total, Hkv, D, device="cuda", dtype=torch.bfloat16) if c["k_out"] else None}
    if c["op"] == "window":
        rows, keys = _window_lengths(c)
        nq, nk = c["rows"] + c["behind"], sum(keys) + c["behind"]
        if c["packed"]:
            buf = rand(nq, (H + 2 * Hkv) * D)
            q, k, v = buf[:, :H * D], buf[:, H * D:(H + Hkv) * D], buf[:, (H + Hkv) * D:]
        else:
            q, k, v = rand(nq, H * D), rand(nk, Hkv * D, std=1.3), rand(nk, Hkv * D)
        ends = [torch.tensor([0] + n, dtype=torch.int32).cumsum(0).to(torch.int32).cuda() for n in (rows, keys)]
        return {"case": c, "q": q, "k": k, "v": v, "cu_q": ends[0], "cu_k": ends[1],
                "out": torch.zeros(nq, H, D, device="cuda", dtype=torch.bfloat16), "lse": torch.zeros(nq, H, device="cuda")}
    lens = _decode_lengths(c)
    state = {"case": c, "q": rand(c["seqs"], H * D), "cache": _handle(_cache(c, g, c["seqs"], c["longest"], True)),
             "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "out": torch.empty(c["seqs"], H, D, device="cuda", dtype=torch.bfloat16), "lse": torch.empty(c["seqs"], H, device="cuda")}
    if own:
        import miroxen_b200 as mx
        state["workspace"] = mx.attn_decode_workspace(state["cache"], H)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"append": _plain_append, "window": _plain_window, "decode": _plain_decode}[c["op"]](s, c)


def _own(s, c):
    import miroxen_b200 as mx
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if c["op"] == "append":
        cache = s["cache"]
        mx.qkv_norm_rope_append(s["q"], s["k"], s["v"], s["q"].shape[0], H, D, s["wq"], s["wk"], 1e-6, s["cos"], s["sin"], s["cos"].shape[0],
                                c["rot"], c["mode"], cache, s["pos"], s["q_out"], seq_ids=s["ids"], k_out=s["k_out"],
                                q_stride=s["q"].stride(0), k_stride=s["k"].stride(0), v_stride=s["v"].stride(0))
        return [s["q_out"], cache.k, cache.v] + ([s["k_out"]] if c["k_out"] else [])
    if c["op"] == "window":
        mx.attn_window(s["q"], s["k"], s["v"], s["q"].shape[0], s["k"].shape[0], H, Hkv, D, D ** -0.5, s["out"], left=c["left"], right=c["right"],
                       sinks=c["sinks"], cu_q=s["cu_q"], cu_k=s["cu_k"], q_stride=s["q"].stride(0), k_stride=s["k"].stride(0),
                       v_stride=s["v"].stride(0), lse=s["lse"])
        return [s["out"], s["lse"]]
    mx.attn_decode_paged(s["q"], s["cache"], s["lens"], H, D ** -0.5, s["out"], left=c["left"], sinks=c["sinks"], lse=s["lse"],
                         workspace=s["workspace"])
    return [s["out"], s["lse"]]


def _norm_rope(x, w, cos, sin, rot, mode):
    """x [rows, heads, D] in 32 bits; cos and sin [rows, 1, rot / 2]."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if mode == INTERLEAVED else (x[..., :rot // 2], x[..., rot // 2:rot])
    turned = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack(turned, -1).flatten(-2) if mode == INTERLEAVED else torch.cat(turned, -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _store(cache, scale, page, slot, x):
    if scale is not None:
        x = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype).view(torch.uint8)
        cache.view(torch.uint8)[page, slot] = x
    else:
        cache[page, slot] = x.to(cache.dtype)


def _plain_append(s, c):
    k_cache, v_cache, table, k_scale, v_scale = s["cache"]
    total = s["q"].shape[0]
    at = (s["ids"] >= 0).nonzero()[:, 0]
    ids, pos = s["ids"][at].long(), s["pos"][at].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _norm_rope(s["q"][at].float().view(-1, c["H"], c["D"]), s["wq"], cos, sin, c["rot"], c["mode"])
    k = _norm_rope(s["k"][at].float().view(-1, c["Hkv"], c["D"]), s["wk"], cos, sin, c["rot"], c["mode"])
    v = s["v"][at].float().view(-1, c["Hkv"], c["D"])
    page, slot = table[ids, pos // c["page"]].long(), pos % c["page"]
    _store(k_cache, k_scale, page, slot, k)
    _store(v_cache, v_scale, page, slot, v)
    s["q_out"][at] = q.to(torch.bfloat16)
    if not c["k_out"]:
        return [s["q_out"], k_cache, v_cache]
    s["k_out"][at] = k.to(torch.bfloat16)
    return [s["q_out"], k_cache, v_cache, s["k_out"]]


def _softmax_product(score, v):
    """score [..., rows, keys] with -inf where a key is not seen; rows that see nothing give 0 and -inf."""
    m = score.amax(-1, keepdim=True)
    p = score.sub_(m.clamp(min=torch.finfo(torch.float32).min)).exp_()
    total = p.sum(-1, keepdim=True)
    return (p @ v) / total.clamp(min=1e-30), (m + total.log())[..., 0]


def _plain_window(s, c):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    nq, nk = s["q"].shape[0], s["k"].shape[0]
    q = s["q"].float().view(nq, H, D).transpose(0, 1)
    k, v = (t.float().view(nk, Hkv, D).transpose(0, 1).repeat_interleave(H // Hkv, 0) for t in (s["k"], s["v"]))
    row, key = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
    seq_q, seq_k = torch.bucketize(row, s["cu_q"][1:].long(), right=True), torch.bucketize(key, s["cu_k"][1:].long(), right=True)
    first_q, first_k = (torch.cat([t.long(), t[-1:].long()]) for t in (s["cu_q"][:-1], s["cu_k"][:-1]))
    more = torch.cat([s["cu_k"].diff() - s["cu_q"].diff(), s["cu_k"][:1]])
    p, j = (row - first_q[seq_q] + more[seq_q])[:, None], (key - first_k[seq_k])[None]
    there = seq_q < c["seqs"]
    seen = (seq_q[:, None] == seq_k[None]) & there[:, None]
    if c["right"] >= 0:
        seen &= j <= p + c["right"]
    if c["left"] >= 0:
        seen &= (j >= p - c["left"]) | (j < c["sinks"])
    score = (q * D ** -0.5) @ k.transpose(1, 2)
    out, lse = _softmax_product(score.masked_fill_(~seen, -math.inf), v)
    out, lse = out.transpose(0, 1).to(torch.bfloat16), lse.transpose(0, 1)
    return [torch.where(there[:, None, None], out, s["out"]), torch.where(there[:, None], lse, s["lse"])]


def _plain_decode(s, c):
    H, Hkv, D, n = c["H"], c["Hkv"], c["D"], c["seqs"]
    k_cache, v_cache, table, k_scale, v_scale = s["cache"]
    k, v = (t.view(torch.uint8 if t.dtype.itemsize == 1 else t.dtype)[table.long()].view(t.dtype).flatten(1, 2).transpose(1, 2).float()
            for t in (k_cache, v_cache))  # [sequences, key heads, tokens, D]
    if k_scale is not None:
        k, v = k.mul_(k_scale[:, None, None]), v.mul_(v_scale[:, None, None])
    q = s["q"].float().view(n, Hkv, H // Hkv, D) * D ** -0.5
    j, last = torch.arange(k.shape[2], device="cuda")[None], s["lens"][:, None].long() - 1
    seen = j <= last
    if c["left"] >= 0:
        seen &= (j >= last - c["left"]) | (j < c["sinks"])
    score = q @ k.transpose(2, 3)
    out, lse = _softmax_product(score.masked_fill_(~seen[:, None, None], -math.inf), v)
    return [out.reshape(n, H, D).to(torch.bfloat16), lse.reshape(n, H)]


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    return {"append": _exact_append, "window": _exact_window, "decode": _exact_decode}[c["op"]](s, c)


def _parts(cache):
    return (cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale) if hasattr(cache, "page_table") else cache


def _exact_append(s, c):
    """The rotation as a product of complex numbers. The cache is given where it is not held in 8 bits."""
    k_cache, v_cache, table, k_scale, _ = _parts(s["cache"])
    half, rot = c["rot"] // 2, c["rot"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    live = s["ids"] >= 0

    def one(x, w, heads):
        x = x.double().reshape(-1, heads, c["D"])
        x = x / (x.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt() * w.double()
        pairs = x[..., :rot].unflatten(-1, (half, 2) if c["mode"] == INTERLEAVED else (2, half))
        axis = -1 if c["mode"] == INTERLEAVED else -2
        z = torch.complex(pairs.select(axis, 0).contiguous(), pairs.select(axis, 1).contiguous()) * turn[s["pos"].long()][:, None, :]
        x[..., :rot] = torch.stack((z.real, z.imag), axis).flatten(-2)
        return x

    q, k = one(s["q"], s["wq"], c["H"]), one(s["k"], s["wk"], c["Hkv"])
    q = torch.where(live[:, None, None], q, 0)
    outs = [q, None, None]
    if k_scale is None:
        v = s["v"].double().reshape(-1, c["Hkv"], c["D"])
        flat = (table.long()[s["ids"].clamp(min=0).long(), (s["pos"] // c["page"]).long()] * c["page"] + s["pos"] % c["page"])[live]
        for i, (x, t) in enumerate(((k, k_cache), (v, v_cache))):
            outs[1 + i] = torch.zeros(t.shape[0] * c["page"], *t.shape[2:], dtype=torch.float64, device="cuda").index_copy_(0, flat, x[live]).view(t.shape)
    return outs + ([torch.where(live[:, None, None], k, 0)] if c["k_out"] else [])


def _exact_rows(q, k, v, scale, see):
    """q [rows, D], k and v [keys, D], see [rows, keys]: from the definition, with logaddexp for the sums."""
    t = torch.where(see, scale * torch.einsum("id,jd->ij", q, k), -math.inf)
    lse = torch.logsumexp(t, 1)
    w = torch.where(see, torch.exp(t - torch.where(lse.isinf(), 0, lse)[:, None]), 0)
    return torch.einsum("ij,jd->id", w, v), lse


def _exact_window(s, c):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    out, lse = s["out"].double(), s["lse"].double()
    q, k, v = (s[n].reshape(s[n].shape[0], -1, D) for n in "qkv")
    at_q = at_k = 0
    for nq, nk in zip(*_window_lengths(c)):
        for r0 in range(0, nq, 2048):
            r1 = min(nq, r0 + 2048)
            p = torch.arange(r0, r1, device="cuda")[:, None] + (nk - nq)
            j = torch.arange(nk, device="cuda")[None, :]
            see = torch.ones(r1 - r0, nk, dtype=torch.bool, device="cuda")
            if c["right"] >= 0:
                see &= j - p <= c["right"]
            if c["left"] >= 0:
                see &= (p - j <= c["left"]) | (j < c["sinks"])
            for h in range(H):
                g = h // (H // Hkv)
                o, l = _exact_rows(q[at_q + r0:at_q + r1, h].double(), k[at_k:at_k + nk, g].double(), v[at_k:at_k + nk, g].double(), D ** -0.5, see)
                out[at_q + r0:at_q + r1, h], lse[at_q + r0:at_q + r1, h] = o, l
        at_q, at_k = at_q + nq, at_k + nk
    return [out, lse]


def _exact_decode(s, c):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    k_cache, v_cache, table, k_scale, v_scale = _parts(s["cache"])
    out = torch.zeros(c["seqs"], H, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(c["seqs"], H, dtype=torch.float64, device="cuda")
    q = s["q"].double().reshape(c["seqs"], Hkv, H // Hkv, D)
    for b, n in enumerate(_decode_lengths(c)):
        j = torch.arange(n, device="cuda")
        if c["left"] >= 0:
            j = j[(n - 1 - j <= c["left"]) | (j < c["sinks"])]
        page = table[b].long()[j // c["page"]]
        kv = [(t.view(torch.uint8)[page, j % c["page"]].view(t.dtype) if t.dtype.itemsize == 1 else t[page, j % c["page"]]).double()
              for t in (k_cache, v_cache)]
        for g in range(Hkv):
            ks, vs = (1.0, 1.0) if k_scale is None else (k_scale[g].double(), v_scale[g].double())
            see = torch.ones(H // Hkv, len(j), dtype=torch.bool, device="cuda")
            o, l = _exact_rows(q[b, g], kv[0][:, g] * ks, kv[1][:, g] * vs, D ** -0.5, see)
            out[b, g * (H // Hkv):(g + 1) * (H // Hkv)], lse[b, g * (H // Hkv):(g + 1) * (H // Hkv)] = o, l
    return [out, lse]
