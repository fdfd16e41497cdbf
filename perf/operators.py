"""What is measured of the attention path around the 4-bit paged key/value cache: the cases, their
inputs, the operators' plain forms in elementary torch operations, the calls a user makes of the
package's own, and the values in 64 bits.

A cached value is ``offset + scale * code`` with a 4-bit code and an fp16 (scale, offset) pair for
each token, kv head and group of ``group`` channels. Sixteen tokens of one kv head make a block of
``16 * (D + 8 * D / group)`` bytes: key codes ``[16, D / 2]`` (channel 2i in the low nibble of byte
i), value codes, the keys' pairs ``[16, D / group, 2]``, the values' pairs. A page is
``page / 16`` blocks of each kv head; the pool is ``[layers, pages, kv_heads, page bytes]``.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
LIMIT = 65504.0   # largest finite fp16: values beyond it are stored as it


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "w4a16-dequant-fused-matmul-kernel_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import w4a16

    return w4a16


# ---------------------------------------------------------------------------------------- cases
# 32 query / 8 kv heads of 128 make the 4096 features, 64 / 8 the 8192 features of the repository's
# layers; 28 / 4 and 16 / 16 stand for groups that are no power of two and for no sharing at all.
def listed():
    return [
        # a prompt's queries and keys on their way to attention
        dict(name="rope prompt", op="rope", tokens=4096, heads=32, kv=8, dim=128, dtype="f16", rot=128, axes=1,
             norm=True, pairs=False),
        # image and video tokens: time, height and width rotate their own channels; part of the head rotates
        dict(name="rope three axes", op="rope", tokens=1037, heads=28, kv=4, dim=128, dtype="bf16", rot=96, axes=3,
             norm=True, pairs=True),
        # one decode step of one sequence: latency
        dict(name="append token", op="append", tokens=1, heads=32, kv=8, dim=128, dtype="f16", rot=128, axes=1,
             norm=True, pairs=False, page=64, group=128),
        # a long prompt into the cache
        dict(name="append prompt", op="append", tokens=8192, heads=64, kv=8, dim=128, dtype="bf16", rot=128, axes=1,
             norm=True, pairs=False, page=32, group=64),
        # one token of one short conversation: latency
        dict(name="attend token", op="attend", seqs=1, new=1, length=777, spread=0.0, idle=0, heads=32, kv=8, dim=128,
             dtype="f16", page=16, group=128, window=0),
        # a decode step of a full batch, lengths all over the place, three slots of the batch unused
        dict(name="attend batch", op="attend", seqs=64, new=1, length=8000, spread=0.9, idle=3, heads=64, kv=8, dim=128,
             dtype="f16", page=64, group=128, window=0),
        # few very long conversations
        dict(name="attend long", op="attend", seqs=2, new=1, length=131071, spread=0.3, idle=0, heads=32, kv=8,
             dim=128, dtype="bf16", page=64, group=64, window=0),
        # five drafted tokens of each sequence checked at once, window attention, heads of 64, no shared heads
        dict(name="attend draft", op="attend", seqs=24, new=5, length=3001, spread=0.6, idle=0, heads=16, kv=16, dim=64,
             dtype="bf16", page=32, group=64, window=1024),
        # prompts in chunks: ragged new tokens behind what is cached already
        dict(name="attend prompt", op="attend", seqs=3, new=4096, length=8192, spread=0.5, idle=0, heads=32, kv=8,
             dim=128, dtype="f16", page=64, group=128, window=0),
        # a few pages moved: latency
        dict(name="pages copy", op="copy", layers=4, pages=64, moved=3, kv=8, dim=128, page=64, group=128),
        # a pool with holes made dense
        dict(name="pages compact", op="compact", layers=16, pages=1200, moved=400, kv=8, dim=128, page=64, group=128,
             seqs=64),
        # parents branch into children, each with its own copy of the last page; finished branches go
        dict(name="pages fork", op="fork", layers=32, pages=2048, moved=48, kv=8, dim=128, page=32, group=128, seqs=96),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "attend", "copy", "compact", "fork"])
    heads, kv = rng.choice([(32, 8), (64, 8), (28, 4), (16, 16), (8, 1), (40, 8), (12, 4)])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["f16", "bf16"])
    group = rng.choice([64, dim])
    page = rng.choice([16, 32, 64, 128])
    if op in ("rope", "append"):
        c = dict(op=op, tokens=_log(rng, 1, 8192), heads=heads, kv=kv, dim=dim, dtype=dtype,
                 rot=rng.choice([dim, dim // 2]), axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.8,
                 pairs=rng.random() < 0.3)
        return dict(c, page=page, group=group) if op == "append" else c
    if op == "attend":
        seqs = _log(rng, 1, 200)
        new = rng.choice([1, 1, _log(rng, 2, 12), _log(rng, 16, 4096)])
        if new > 12:
            seqs = rng.randint(1, 2)
            heads, kv = (heads, kv) if heads <= 32 else (32, 8)
        length = _log(rng, new, 8192 if new > 12 else max(new, min(131072, 260000 // seqs)))
        return dict(op=op, seqs=seqs, new=new, length=length, spread=rng.choice([0.0, 0.5, 0.9]),
                    idle=rng.choice([0, 0, 1]) if seqs > 2 else 0, heads=heads, kv=kv, dim=dim, dtype=dtype, page=page,
                    group=group, window=rng.choice([0, 0, _log(rng, 1, 4096)]))
    pages = _log(rng, 16, 1200)
    c = dict(op=op, layers=rng.randint(1, 16), pages=pages, moved=max(1, int(pages * rng.uniform(0.02, 0.3))),
             kv=rng.choice([1, 4, 8]), dim=dim, page=page, group=group)
    return c if op == "copy" else dict(c, seqs=rng.randint(2, 96))


# ---------------------------------------------------------------------------------------- sizes
def _block_bytes(c):
    return 16 * (c["dim"] + 8 * (c["dim"] // c["group"]))


def _page_bytes(c):
    return c["page"] // 16 * _block_bytes(c)


def _lens(c):
    """Length and new tokens of each sequence: a plain function of the case. The last `idle` are unused slots
    (length 0); the longer `spread`, the more the lengths differ. A prompt's new tokens differ likewise."""
    lens, new = [], []
    for i in range(c["seqs"]):
        part = 1.0 - c["spread"] * ((i * 0.6180339887) % 1.0)
        n = c["new"] if c["new"] <= 12 else max(1, int(c["new"] * part))
        lens.append(0 if i >= c["seqs"] - c["idle"] else max(n, int(c["length"] * part)))
        new.append(n)
    return lens, new


def _pairs_and_tokens(c):
    """(query token, cached token) pairs that attend, and cached tokens that some query sees, of a kv head."""
    pairs = seen = 0
    for n, q in zip(*_lens(c)):
        w = c["window"] if c["window"] else 1 << 40
        if n == 0:
            continue
        for_each = np.minimum(np.arange(n - q + 1, n + 1, dtype=np.int64), w)
        pairs += int(for_each.sum())
        seen += min(n, q - 1 + w)
    return pairs, seen


def work(case):
    c = case
    if c["op"] in ("rope", "append"):
        t, d = c["tokens"], c["dim"]
        qk = t * (c["heads"] + c["kv"]) * d * 2
        side = t * c["axes"] * 8 + t * c["rot"] * 4 + 4 * d
        if c["op"] == "rope":
            return {"bytes": 2 * qk + side, "flops": 8 * qk // 2}
        v = t * c["kv"] * d * 2
        cache = t * c["kv"] * (_block_bytes(c) // 16)
        # queries, keys and values in; queries, the cache's tokens, and those read back out
        return {"bytes": qk + v + side + t * 8 + t * c["heads"] * d * 2 + cache + 2 * v,
                "flops": 8 * qk // 2 + 8 * v}
    if c["op"] == "attend":
        pairs, seen = _pairs_and_tokens(c)
        rows = sum(_lens(c)[1]) * c["heads"]
        return {"bytes": seen * c["kv"] * (_block_bytes(c) // 16) + rows * c["dim"] * 4 + rows * 4 + 4 * seen // c["page"],
                "flops": 4 * c["dim"] * c["heads"] * pairs}
    moved = 2 * _moved(c) * c["layers"] * c["kv"] * _page_bytes(c)
    if c["op"] == "copy":
        return {"bytes": moved + 8 * _moved(c), "flops": 0}
    if c["op"] == "compact":
        return {"bytes": moved + 2 * 4 * (c["pages"] + c["seqs"] * _table_width(c)), "flops": 0}
    return {"bytes": moved + 2 * 4 * (c["pages"] + c["seqs"] * _table_width(c) + c["seqs"]), "flops": 0}


def _table_width(c):
    return max(4, -(-2 * c["pages"] // c["seqs"]))


def _parents(c):
    return max(1, min(c["seqs"] // 4, c["pages"] // 4))


def _moved(c):
    """Pages whose bytes move: as many as asked for that the pool and the tables allow."""
    if c["op"] == "copy":
        return min(c["moved"], c["pages"] // 2)
    if c["op"] == "compact":
        return min(c["moved"], c["pages"] - c["pages"] * 5 // 8)
    return min(c["moved"], c["seqs"] - _parents(c), c["pages"] // 4)


# --------------------------------------------------------------------------------------- inputs
def _dtype(c):
    return torch.float16 if c["dtype"] == "f16" else torch.bfloat16


def _cos_sin(n, rot, base=10000.0):
    f = base ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float32) / rot)
    a = torch.arange(n, device=DEV, dtype=torch.float32)[:, None] * f
    return torch.cat([a.cos(), a.sin()], -1)


def _quantise(x, group):
    """fp32 [..., D] -> codes uint8 [..., D], (scale, offset) fp16 [..., D / group, 2]."""
    x = x.unflatten(-1, (-1, group)).clamp(-LIMIT, LIMIT)
    offset = x.amin(-1).half()
    scale = ((x.amax(-1) - offset.float()) / 15.0).half()
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    steps = (x - offset.float()[..., None]) * (1.0 / scale.float())[..., None]
    codes = steps.round().clamp(0, 15).to(torch.uint8)
    return codes.flatten(-2), torch.stack([scale, offset], -1)


def _fill_pool(g, c, layers, pages):
    """A pool whose every block holds keys and values as a model makes them, quantised."""
    d, kv = c["dim"], c["kv"]
    pool = torch.empty((layers, pages, kv, c["page"] // 16, _block_bytes(c)), device=DEV, dtype=torch.uint8)
    tilt = torch.randn((2, kv, 1, 1, d), generator=g, device=DEV) * 0.5
    step = max(1, (1 << 26) // (kv * c["page"] * d))
    for layer in range(layers):
        for at in range(0, pages, step):
            n = min(step, pages - at)
            for which in (0, 1):
                x = torch.randn((n, kv, c["page"] // 16, 16, d), generator=g, device=DEV) * (1.0 + which)
                codes, pairs = _quantise(x + tilt[which], c["group"])
                part = pool[layer, at:at + n]
                part[..., which * 8 * d:(which + 1) * 8 * d] = (codes[..., 0::2] | (codes[..., 1::2] << 4)).flatten(-2)
                size = 64 * (d // c["group"])
                lo = 16 * d + which * size
                part[..., lo:lo + size] = pairs.flatten(-4).view(torch.uint8).view(n, kv, c["page"] // 16, size)
    return pool.flatten(-2)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    s = {"case": c}
    d = c["dim"]
    if c["op"] in ("rope", "append"):
        t, dt = c["tokens"], _dtype(c)
        width = (c["heads"] + 2 * c["kv"]) * d
        qkv = (torch.randn((t, width), generator=g, device=DEV) * 2.0).to(dt)
        q, k, v = qkv.split([c["heads"] * d, c["kv"] * d, c["kv"] * d], 1)   # views of the projection's output
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in (q, k, v))
        s["wq"] = s["wk"] = None
        if c["norm"]:
            s["wq"], s["wk"] = ((1.0 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(dt) for _ in range(2))
        first = int(host.randint(0, 20000))
        pos = first + torch.arange(t, device=DEV)
        if c["axes"] == 3:
            pos = torch.stack([pos, first + torch.arange(t, device=DEV) // 24 % 24, first + torch.arange(t, device=DEV) % 24])
            third = c["rot"] // 2 // 3
            s["sections"] = (c["rot"] // 2 - 2 * third, third, third)
        else:
            s["sections"] = None
        s["pos"] = pos.contiguous()
        s["cos_sin"] = _cos_sin(32768, c["rot"])
        if c["op"] == "append":
            pages = 2 * -(-t // c["page"]) + 3
            order = torch.from_numpy(host.permutation(pages)).to(DEV)
            at = torch.arange(t, device=DEV) + int(host.randint(0, c["page"]))
            s["slots"] = order[at // c["page"]] * c["page"] + at % c["page"]
            s["pool"] = torch.zeros((1, pages, c["kv"], _page_bytes(c)), device=DEV, dtype=torch.uint8)
            s["dtype"] = dt
    elif c["op"] == "attend":
        lens, new = _lens(c)
        need = [-(-n // c["page"]) for n in lens]
        pages = sum(need) + 2
        s["pool"] = _fill_pool(g, c, 1, pages)
        order = host.permutation(pages)
        table = np.zeros((c["seqs"], max(max(need), 1)), np.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        s["table"] = torch.from_numpy(table).to(DEV)
        s["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
        heat = 0.5 * 6.0 ** torch.rand((1, c["heads"], 1), generator=g, device=DEV)   # flat and peaked heads
        s["q"] = (torch.randn((sum(new), c["heads"], d), generator=g, device=DEV) * heat).to(_dtype(c))
        s["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), device=DEV, dtype=torch.int32)
        s["most"] = max(new)
    else:
        s["pool"] = torch.randint(0, 256, (c["layers"], c["pages"], c["kv"], _page_bytes(c)), generator=g, device=DEV,
                                  dtype=torch.uint8)
        order = host.permutation(c["pages"]).astype(np.int32)
        if c["op"] == "copy":
            m = _moved(c)
            s["src"], s["dst"] = (torch.from_numpy(x.copy()).to(DEV) for x in (order[:m], order[m:2 * m]))
        else:
            s.update(_tables(c, host, order))
    if own and "pool" in s:
        w = _package()
        s["cache"] = w.KV4Cache(s["pool"].shape[0], s["pool"].shape[1], c["kv"], d, page_size=c["page"],
                                group_size=c["group"], pool=s["pool"])
        if "refs" in s:
            s["pages"] = w.KV4Pages(s["refs"], s["table"], s["lens"], c["page"])
    return s


def _tables(c, host, order):
    """Reference counts, block table and lengths of sequences that hold pages all over the pool."""
    width, seqs, page = _table_width(c), c["seqs"], c["page"]
    refs = np.zeros(c["pages"], np.int32)
    table = np.full((seqs, width), -1, np.int32)
    lens = np.zeros(seqs, np.int32)
    if c["op"] == "compact":
        # `live` pages are in use; `m` of them lie beyond the first `live`, and leave as many holes there
        m, live = _moved(c), c["pages"] * 5 // 8
        low, high = host.permutation(live)[:live - m], live + host.permutation(c["pages"] - live)[:m]
        use = host.permutation(np.concatenate([low, high])).astype(np.int32)
        ends = [min(live, live * (i + 1) // seqs) for i in range(seqs)]
        for i, (at, to) in enumerate(zip([0] + ends, ends)):
            table[i, :to - at] = use[at:to]
            lens[i] = max(0, (to - at) * page - int(host.randint(0, page)))
            refs[use[at:to]] += 1
            if i % 3 == 2 and to > at and table[i - 1, 0] >= 0:   # a page that two sequences share
                table[i, to - at] = table[i - 1, 0]
                refs[table[i - 1, 0]] += 1
                lens[i] = (to - at + 1) * page
        out = {"refs": refs, "table": table, "lens": lens}
    else:
        parents, m = _parents(c), _moved(c)
        at = 0
        for i in range(parents):
            n = max(1, min(width, (c["pages"] // 2) // parents))
            table[i, :n] = order[at:at + n]
            lens[i] = n * page - 1 - int(host.randint(0, page - 1))   # the last page is partly filled
            at += n
        refs[order[:at]] = 1
        out = {"refs": refs, "table": table, "lens": lens,
               "parents": np.arange(m, dtype=np.int32) % parents,
               "children": (parents + np.arange(m)).astype(np.int32),
               "gone": np.arange(0, parents, 2, dtype=np.int32)}
    return {k: torch.from_numpy(v).to(DEV) for k, v in out.items()}


# ----------------------------------------------------------------------------------- plain forms
def _norm(x, w, eps):
    x = x.float()
    if w is None:
        return x
    return x * (1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)) * w.float()


def _rotate(x, cos, sin, rot, pairs):
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :rot // 2], r[..., rot // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _angles(s):
    c = s["case"]
    half = c["rot"] // 2
    cs = s["cos_sin"][s["pos"]]
    if s["sections"] is not None:
        axis = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(s["sections"], device=DEV), output_size=half)
        cs = cs.gather(0, torch.cat([axis, axis])[None, None].expand(1, cs.shape[1], -1))[0]
    return cs[:, None, :half], cs[:, None, half:]


def _plain_rope(s):
    c = s["case"]
    cos, sin = _angles(s)
    return tuple(_rotate(_norm(s[x], s["w" + x], 1e-6), cos, sin, c["rot"], c["pairs"]) for x in "qk")


def _regions(pool, c):
    """Views of a layer's pool [pages, kv, page bytes]: key codes, value codes, key pairs, value pairs."""
    d, n = c["dim"], c["dim"] // c["group"]
    b = pool.unflatten(-1, (c["page"] // 16, _block_bytes(c)))
    pairs = b[..., 16 * d:].view(torch.float16).unflatten(-1, (2, 16, n, 2))
    return (b[..., :8 * d].unflatten(-1, (16, d // 2)), b[..., 8 * d:16 * d].unflatten(-1, (16, d // 2)),
            pairs[..., 0, :, :, :], pairs[..., 1, :, :, :])


def _values(codes, pairs, c):
    """What packed codes [..., D / 2] and pairs [..., D / group, 2] stand for, fp32 [..., D]."""
    x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, c["group"]))
    return (x * pairs[..., :1].float() + pairs[..., 1:].float()).flatten(-2)


def _plain_append(s):
    c = s["case"]
    q, k = _plain_rope(s)
    kc, vc, kp, vp = _regions(s["pool"][0], c)
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    for x, codes, pairs in ((k, kc, kp), (s["v"].float(), vc, vp)):
        new, pair = _quantise(x, c["group"])
        codes[page, :, at // 16, at % 16] = new[..., 0::2] | (new[..., 1::2] << 4)
        pairs[page, :, at // 16, at % 16] = pair
    kv = torch.stack([_values(codes[page, :, at // 16, at % 16], pairs[page, :, at // 16, at % 16], c)
                      for codes, pairs in ((kc, kp), (vc, vp))])
    return {"q": q.to(s["dtype"]), "kv": kv.to(s["dtype"])}


def _plain_attend(s):
    c = s["case"]
    d, kv, most = c["dim"], c["kv"], s["most"]
    share = c["heads"] // kv
    seqs, width = s["table"].shape
    kc, vc, kp, vp = (x[s["table"]] for x in _regions(s["pool"][0], c))   # [seqs, width, kv, blocks, 16, ...]
    k, v = (_values(codes, pairs, c).permute(0, 2, 1, 3, 4, 5).reshape(seqs, kv, 1, -1, d)
            for codes, pairs in ((kc, kp), (vc, vp)))
    # queries [seqs, kv, share, most, d], those beyond a sequence's own are any and are left out again
    new = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(most, device=DEV)
    row = (s["cu"][:-1, None] + torch.minimum(i, new[:, None] - 1)).long()
    q = s["q"].float()[row].unflatten(2, (kv, share)).permute(0, 2, 3, 1, 4)
    scores = (q * (1.0 / math.sqrt(d))) @ k.transpose(-1, -2)
    t = torch.arange(k.shape[3], device=DEV)
    last = (s["lens"] - new)[:, None] + i                              # the position of each query
    see = (t <= last[..., None]) & (t < s["lens"][:, None, None])
    if c["window"]:
        see &= t > last[..., None] - c["window"]
    scores = scores.masked_fill(~see[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (torch.log(total) + top)[..., 0]
    back = torch.repeat_interleave(torch.arange(seqs, device=DEV), new, output_size=s["q"].shape[0])
    own_row = torch.arange(s["q"].shape[0], device=DEV) - s["cu"][:-1][back]
    o = o.permute(0, 3, 1, 2, 4)[back, own_row].flatten(1, 2)
    lse = lse.permute(0, 3, 1, 2)[back, own_row].flatten(1, 2)
    return {"o": o.to(s["q"].dtype), "lse": lse}


def _plain_compact(s):
    live = s["refs"] > 0
    count = live.sum()
    pages = torch.arange(live.numel(), device=DEV)
    hole, mover = ~live & (pages < count), live & (pages >= count)
    # the i-th live page beyond `count` goes to the i-th free page before it
    src, dst = mover.nonzero()[:, 0], hole.nonzero()[:, 0]
    s["pool"][:, dst] = s["pool"][:, src]
    to = pages.clone()
    to[src] = dst
    refs = torch.zeros_like(s["refs"])
    refs[to[live]] = s["refs"][live]
    table = torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), s["table"])
    return refs, table


def _plain_fork(s):
    c = s["case"]
    refs, table, lens = s["refs"].clone(), s["table"].clone(), s["lens"].clone()
    par, kid = s["parents"].long(), s["children"].long()
    n = lens[par]
    held, tail = (n + c["page"] - 1) // c["page"], n % c["page"] != 0
    rows = table[par]
    col = torch.arange(table.shape[1], device=DEV)
    # the lowest free pages, in the order of the pairs, for the partly filled last pages
    new = (refs == 0).nonzero()[:, 0].int()
    own_page = torch.where(tail, new[(tail.cumsum(0) - 1).clamp(min=0)], torch.full_like(n, -1))
    is_tail = tail[:, None] & (col == held[:, None] - 1)
    old = rows.gather(1, (held - 1).clamp(min=0)[:, None].long())[:, 0]
    s["pool"][:, own_page[tail].long()] = s["pool"][:, old[tail].long()]
    rows = torch.where(is_tail, own_page[:, None], rows)
    held_here = col < held[:, None]
    refs.index_add_(0, rows[held_here].long(), torch.ones_like(rows[held_here]))
    table[kid] = torch.where(held_here, rows, torch.full_like(rows, -1))
    lens[kid] = n
    # the branches that are finished
    gone = s["gone"].long()
    rows = table[gone]
    used = rows[rows >= 0]
    refs.index_add_(0, used.long(), -torch.ones_like(used))
    table[gone] = -1
    lens[gone] = 0
    return refs, table, lens


def run(state):
    s = state
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "rope":
            return {x: y.to(s["q"].dtype) for x, y in zip("qk", _plain_rope(s))}
        if op == "append":
            return _plain_append(s)
        if op == "attend":
            return _plain_attend(s)
        if op == "copy":
            s["pool"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
            return {"pool": s["pool"].view(torch.int32)}
        if op == "compact":
            refs, table = _plain_compact(s)
            return {"pool": s["pool"].view(torch.int32), "refs": refs, "table": table}
        refs, table, lens = _plain_fork(s)
        return {"pool": s["pool"].view(torch.int32), "refs": refs, "table": table, "lens": lens}
    w = _package()
    if op == "rope":
        q, k = w.qk_norm_rope(s["q"], s["k"], s["pos"], s["cos_sin"], s["wq"], s["wk"], sections=s["sections"],
                              interleaved=c["pairs"])
        return {"q": q, "k": k}
    if op == "append":
        q = w.qk_norm_rope_append(s["q"], s["k"], s["v"], s["cache"], 0, s["slots"], s["pos"], s["cos_sin"], s["wq"],
                                  s["wk"], sections=s["sections"], interleaved=c["pairs"])
        return {"q": q, "kv": w.kv4_gather(s["cache"], 0, s["slots"], s["dtype"])}
    if op == "attend":
        o, lse = w.kv4_attention(s["q"], s["cache"], 0, s["table"], s["lens"], cu_q=s["cu"], max_q=s["most"],
                                 window=c["window"], return_lse=True)
        return {"o": o, "lse": lse}
    if op == "copy":
        w.kv4_copy_pages(s["cache"], s["src"], s["dst"])
        return {"pool": s["pool"].view(torch.int32)}
    if op == "compact":
        pages = w.kv4_compact(s["cache"], s["pages"])
        return {"pool": s["pool"].view(torch.int32), "refs": pages.refs, "table": pages.block_table}
    pages, _ = w.kv4_fork(s["cache"], s["pages"], s["parents"], s["children"])
    w.kv4_release(pages, s["gone"], out=pages)
    return {"pool": s["pool"].view(torch.int32), "refs": pages.refs, "table": pages.block_table, "lens": pages.kv_lens}


# ------------------------------------------------------------------------------ values in 64 bits
def _exact_head(x, w, pos, c, sections):
    """x [tokens, heads, D] float64 normed, weighted, and each pair of channels turned by its own angle. The
    angles' cosines and sines are inputs (an fp32 table), so they are taken as they are given."""
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + 1e-6) * w.double()
    half = c["rot"] // 2
    cs = _cos_sin(32768, c["rot"]).double()
    out = x.clone()
    for i in range(half):
        p = pos
        if sections is not None:
            p = pos[0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2]
        co, si = cs[p, i][:, None], cs[p, half + i][:, None]
        a, b = (2 * i, 2 * i + 1) if c["pairs"] else (i, half + i)
        out[..., a] = x[..., a] * co - x[..., b] * si
        out[..., b] = x[..., b] * co + x[..., a] * si
    return out


def _exact_cached(x, c):
    """x float64 as the cache holds it."""
    out = torch.empty_like(x)
    for lo in range(0, c["dim"], c["group"]):
        y = x[..., lo:lo + c["group"]].clamp(-LIMIT, LIMIT)
        off = y.min(-1, keepdim=True).values.half().double()
        sc = ((y.max(-1, keepdim=True).values - off) / 15).half().double()
        sc[sc <= 0] = 1.0
        out[..., lo:lo + c["group"]] = torch.clamp(torch.round((y - off) / sc), 0, 15) * sc + off
    return out


def _exact_tokens(s, i, n):
    """Keys and values of a sequence's first n tokens, float64 [kv, n, D] each, from the pool's bytes."""
    c = s["case"]
    d, groups = c["dim"], c["dim"] // c["group"]
    need = -(-n // c["page"])
    b = s["pool"][0, s["table"][i, :need].long()]                           # [need, kv, page bytes]
    b = b.view(need, c["kv"], c["page"] // 16, _block_bytes(c)).transpose(0, 1).reshape(c["kv"], -1, _block_bytes(c))
    out = []
    for which in (0, 1):
        words = b[..., which * 8 * d:(which + 1) * 8 * d].contiguous().view(torch.int32).view(c["kv"], -1, 16, d // 8)
        codes = torch.stack([(words >> (4 * j)) & 15 for j in range(8)], -1).reshape(c["kv"], -1, d).double()
        lo = 16 * d + which * 64 * groups
        pair = b[..., lo:lo + 64 * groups].contiguous().view(torch.float16).view(c["kv"], -1, groups, 2).double()
        out.append((codes * pair[..., 0].repeat_interleave(c["group"], -1) + pair[..., 1].repeat_interleave(c["group"], -1))[:, :n])
    return out


def exact(case, seed):
    c = case
    if c["op"] in ("copy", "compact", "fork"):
        return None   # whole numbers only
    s = prepare(c, seed)
    if c["op"] in ("rope", "append"):
        q = _exact_head(s["q"].double(), s["wq"], s["pos"], c, s["sections"])
        k = _exact_head(s["k"].double(), s["wk"], s["pos"], c, s["sections"])
        if c["op"] == "rope":
            return {"q": q, "k": k}
        return {"q": q, "kv": torch.stack([_exact_cached(k, c), _exact_cached(s["v"].double(), c)])}
    lens, new = _lens(c)
    share = c["heads"] // c["kv"]
    o = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    lse = torch.full(s["q"].shape[:2], -math.inf, device=DEV, dtype=torch.float64)
    first = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        if n:
            k, v = _exact_tokens(s, i, n)
            for lo in range(0, m, 512):
                hi = min(m, lo + 512)
                at = torch.arange(n - m + lo, n - m + hi, device=DEV)[:, None]
                t = torch.arange(n, device=DEV)[None]
                hide = t > at
                if c["window"]:
                    hide |= t <= at - c["window"]
                for h in range(c["heads"]):
                    x = s["q"][first + lo:first + hi, h].double() @ k[h // share].T / math.sqrt(c["dim"])
                    x[hide] = -math.inf
                    lse[first + lo:first + hi, h] = torch.logsumexp(x, -1)
                    o[first + lo:first + hi, h] = torch.softmax(x, -1) @ v[h // share]
        first += m
    return {"o": o, "lse": lse}
