"""The operators of the paged context cache: what a policy's VLM does with its tokens beside the action expert.

A step of such a server appends the new tokens of many requests (prompts, camera frames, answered tokens) to a paged
K/V cache and attends from them:

  map     block tables and slots of the step's tokens, made on the GPU from the requests' lengths (``PagePool.map``)
  rope    the multi-axis rotary of the tokens' q and k, with per-head norms where the model has them, k and v stored in
          their pages (``AxesRotary.store``) or returned (``AxesRotary.__call__``, the cross-attention source's form)
  attend  attention of the new tokens over the cache: causal or not, with a sliding window and first tokens that stay
          visible (``page_attend``)

``own`` false: ``run`` computes them from elementary torch operations in 32 bits (angles in 64).
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
THETA, EPS = 1e6, 1e-6
SCORES_MAX = 2.2e9  # entries of the padded score matrix of a plain attention: its temporaries fit the card


def _paged():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reki-megakernel_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mkx import paged
    return paged


# map: B request slots of `cols` pages of P rows, `idle` % of them without new tokens, `ended` % returning their pages; a
# request has up to `old` cached tokens and appends `lo` to `hi`; `spare` token rows behind the last one; `pool` % of the
# pages that the step needs are there.
_MAP = {"op": "map", "B": 16, "P": 64, "lo": 1, "hi": 1, "old": 4096, "idle": 0, "ended": 0, "spare": 0, "pool": 130}
# rope: T tokens, NQ query heads and NK key/value heads of HD, `axes` position axes, positions up to `far`; store: into
# pages of P rows (every 16th token padding); norm: q and k normed per head; fused: q, k, v are views of one projection.
_ROPE = {"op": "rope", "T": 16, "NQ": 16, "NK": 2, "HD": 128, "axes": 3, "far": 32768, "P": 64, "store": True,
         "norm": False, "fused": True, "dtype": "bf16"}
# attend: B requests with lo to hi new tokens each and old_lo to old_hi cached ones before them; `spare` rows of q behind
# the last sequence; single: requests whose chunk is one token, in % (a mixed batch).
_ATT = {"op": "attend", "B": 16, "lo": 1, "hi": 1, "old_lo": 64, "old_hi": 4096, "NQ": 16, "NK": 2, "HD": 128, "P": 64,
        "causal": True, "window": 0, "sinks": 0, "single": 0, "spare": 0, "dtype": "bf16"}


def _case(base, name, **kw):
    return {"name": name, **base, **kw}


def listed():
    return [
        # one answered token of each of sixteen requests: the smallest step, all latency
        _case(_MAP, "map_tokens"),
        # a camera frame's tokens of sixty-four robots, some idle, some whose episode has ended
        _case(_MAP, "map_frames", B=64, lo=200, hi=333, old=8192, idle=20, ended=10, spare=1000),
        # a large mixed step: prompts of very different lengths, with a pool that does not hold the last of them
        _case(_MAP, "map_prompts", B=500, P=16, lo=1, hi=1024, old=2048, idle=5, ended=5, pool=97),
        # sixteen answered tokens: rotary, store
        _case(_ROPE, "rope_tokens"),
        # three cameras of a frame and an instruction, with q and k norms
        _case(_ROPE, "rope_frame", T=1100, norm=True),
        # the keys and queries of eight robots' source contexts in the expert's layout (12 heads of 64), returned
        _case(_ROPE, "rope_source", T=2400, NQ=12, NK=12, HD=64, axes=3, far=1024, store=False, fused=False, dtype="fp16"),
        # a prefill step of long prompts
        _case(_ROPE, "rope_prompts", T=30011, NQ=32, NK=8, axes=1, far=131072, P=16),
        # sixteen answered tokens over short histories: latency
        _case(_ATT, "attend_tokens"),
        # thirty-two answered tokens over long ragged histories: the cache's bytes
        _case(_ATT, "attend_tokens_long", B=32, old_lo=2000, old_hi=32000, NQ=32, NK=8),
        # a frame of eight robots over a window of their last frames, the prompt's first tokens kept
        _case(_ATT, "attend_frames", B=8, lo=200, hi=333, old_lo=1000, old_hi=12000, window=2048, sinks=40, P=16, spare=77),
        # a mixed step of heads of 64 that are not shared: chunks beside single tokens
        _case(_ATT, "attend_mixed", B=24, lo=100, hi=500, single=60, old_lo=0, old_hi=6000, NQ=12, NK=12, HD=64, dtype="fp16"),
        # a prompt of 8192 tokens at once: the matrix products
        _case(_ATT, "attend_prompt", B=1, lo=8192, hi=8192, old_lo=0, old_hi=0, P=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    top = {c["op"]: work(c) for c in listed()}  # the last listed case of an operator is its largest in operations
    top_bytes = work(listed()[8])["bytes"]
    while True:
        op = rng.choice(["map", "map", "rope", "rope", "attend", "attend", "attend", "attend"])
        P = rng.choice([16, 32, 64, 128, 256])
        if op == "map":
            hi = _log_int(rng, 1, 1024)
            c = {**_MAP, "B": _log_int(rng, 1, 500), "P": P, "lo": rng.choice([0, 1, hi]), "hi": hi, "old": _log_int(rng, 1, 8192),
                 "idle": rng.choice([0, 10, 50]), "ended": rng.choice([0, 0, 20]), "spare": rng.choice([0, rng.randint(1, 2000)]),
                 "pool": rng.choice([100, 130, 130, 80])}
        elif op == "rope":
            NK = rng.choice([1, 2, 4, 8])
            c = {**_ROPE, "T": _log_int(rng, 1, 30000), "NK": NK, "NQ": NK * rng.randint(1, 32 // NK), "HD": rng.choice([64, 128]),
                 "axes": rng.choice([1, 2, 3, 3]), "far": _log_int(rng, 1000, 1 << 20), "P": P, "store": rng.random() < 0.7,
                 "norm": rng.random() < 0.5, "fused": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16"])}
        else:
            NK = rng.choice([1, 2, 4, 8, 12])
            hi = rng.choice([1, _log_int(rng, 1, 8192), _log_int(rng, 1, 8192), _log_int(rng, 2, 600)])
            old = _log_int(rng, 1, 32000)
            causal = rng.random() < 0.8
            window = rng.choice([0, 0, _log_int(rng, 1, 4096)]) if causal else 0
            c = {**_ATT, "B": _log_int(rng, 1, 64), "lo": rng.choice([1, hi, max(1, hi // 2)]), "hi": hi, "old_lo": rng.choice([0, old // 2, old]),
                 "old_hi": old, "NK": NK, "NQ": NK * rng.randint(1, max(1, 32 // NK)), "HD": rng.choice([64, 128]), "P": P, "causal": causal,
                 "window": window, "sinks": rng.choice([0, 4, rng.randint(1, 128)]) if window else 0,
                 "single": rng.choice([0, 0, 50]), "spare": rng.choice([0, rng.randint(1, 100)]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
            if c["B"] * c["NQ"] * hi * (old + hi) > SCORES_MAX / 2:
                continue
        w = work(c)
        if w["flops"] <= top[op]["flops"] and w["bytes"] <= max(top[op]["bytes"], top_bytes if op == "attend" else 0):
            return c


# ---- lengths, on the host as a server's scheduler holds them: the case gives the requests, the seed their order ----------

def _lens(c, seed):
    """(new tokens, cached tokens before them, ended) of each request, as lists."""
    g = torch.Generator().manual_seed(sum(ord(x) * 31 ** i for i, x in enumerate(repr(sorted(c.items())))) % (1 << 40))
    B = c["B"]
    add = torch.randint(c["lo"], c["hi"] + 1, (B,), generator=g)
    if c["op"] == "map":
        old = torch.randint(0, c["old"] + 1, (B,), generator=g)
        add = torch.where(torch.rand(B, generator=g) * 100 < c["idle"], 0, add)
    else:
        old = torch.randint(c["old_lo"], c["old_hi"] + 1, (B,), generator=g)
        add = torch.where(torch.rand(B, generator=g) * 100 < c["single"], 1, add)
    ended = (torch.rand(B, generator=g) * 100 < c.get("ended", 0)).int()
    order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
    return add[order].tolist(), old[order].tolist(), ended[order].tolist()


def _cdiv(a, b):
    return -(-a // b)


def _visible(p, n, c):
    """Keys that the query at position p of a request of n tokens sees."""
    if not c["causal"]:
        return n
    return p + 1 if not c["window"] or p < c["window"] else c["window"] + min(c["sinks"], p + 1 - c["window"])


def _visible_sum(p0, q, n, c):
    """The sum of _visible over the q positions from p0 on."""
    if not c["causal"]:
        return q * n
    tri = lambda a, b: (a + b) * (b - a + 1) // 2 if b >= a else 0  # noqa: E731 a + (a + 1) + ... + b
    W, S, end = c["window"] or p0 + q, c["sinks"], p0 + q
    full = tri(p0 + 1, min(end, W))
    part = tri(max(p0, W) + 1 - W, min(end - W, S)) if end > W else 0  # sinks seen one more by one more
    rest = max(0, end - max(p0, W, W + S)) * S
    return full + max(0, end - max(p0, W)) * W + part + rest


def work(c):
    """Bytes and operations of one pass for the mean lengths: inputs read once, outputs written once."""
    if c["op"] == "map":
        tokens = c["B"] * (c["lo"] + c["hi"]) / 2 * (1 - c["idle"] / 100) + c["spare"]
        pages = tokens / c["P"] + c["B"]
        return {"bytes": tokens * 12 + c["B"] * 28 + pages * 8, "flops": tokens}
    if c["op"] == "rope":
        heads = 2 * (c["NQ"] + c["NK"]) + (2 * c["NK"] if c["store"] else 0)
        return {"bytes": c["T"] * (heads * c["HD"] * 2 + c["axes"] * 4 + (8 if c["store"] else 0)),
                "flops": c["T"] * (c["NQ"] + c["NK"]) * c["HD"] * (7 if c["norm"] else 3)}
    share = c["single"] / 100
    rows = pairs = keys = 0.0
    for part, q in ((share, 1), (1 - share, (c["lo"] + c["hi"]) // 2)):
        old = (c["old_lo"] + c["old_hi"]) // 2
        rows += part * c["B"] * q
        pairs += part * c["B"] * _visible_sum(old, q, old + q, c)
        keys += part * c["B"] * (min(old + q, c["window"] + q + c["sinks"]) if c["window"] else old + q)
    return {"bytes": (rows * 2 * c["NQ"] + keys * 2 * c["NK"]) * c["HD"] * 2 + keys / c["P"] * 4,
            "flops": 4 * pairs * c["NQ"] * c["HD"]}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _prepare_map(c, seed, dev, g):
    add, old, ended = _lens(c, seed)
    B, P = c["B"], c["P"]
    held = [_cdiv(n, P) for n in old]
    need = sum(_cdiv(n + a, P) - h for n, a, h, e in zip(old, add, held, ended) if not e)
    cols = max(1, max(_cdiv(n + a, P) for n, a in zip(old, add)))
    free = need * c["pool"] // 100
    n_pages = sum(held) + free + 1
    T = max(1, sum(a for a, e in zip(add, ended) if not e) + c["spare"])
    perm = torch.randperm(n_pages, generator=g, device=dev, dtype=torch.int32)
    held_t = torch.tensor(held, device=dev)
    at = torch.arange(cols, device=dev)[None, :] < held_t[:, None]
    table = torch.full((B, cols), -1, dtype=torch.int32, device=dev)
    table[at] = perm[: sum(held)]
    # the free pages wait in a ring queue, somewhere in its middle
    head = int(torch.randint(0, n_pages, (1,), generator=torch.Generator().manual_seed(seed)))
    queue = torch.full((n_pages,), -1, dtype=torch.int32, device=dev)
    queue[(head + torch.arange(free, device=dev)) % n_pages] = perm[sum(held): sum(held) + free]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = {"add": i32(add), "done": i32(ended) if c["ended"] else None, "len": i32(old), "table": table, "queue": queue,
         "ends": i32([head, free]), "T": T, "P": P}
    if own:
        s["pool"] = _paged().PagePool(slots=B, n_pages=n_pages, page_rows=P, table_cols=cols, max_tokens=T, device=dev)
        s["pool"].load_state_dict({k: s[k] for k in ("len", "table", "queue", "ends")})
    return s


def _axis_of(c):
    """The axis of each of the HD / 2 frequencies: sections of equal size, the first axis taking what is left."""
    part = c["HD"] // 2 // (c["axes"] + 1) if c["axes"] > 1 else 0
    sections = [c["HD"] // 2 - part * (c["axes"] - 1)] + [part] * (c["axes"] - 1)
    return [a for a, n in enumerate(sections) for _ in range(n)]


def _prepare_rope(c, seed, dev, g):
    T, NQ, NK, HD, dt = c["T"], c["NQ"], c["NK"], c["HD"], DTYPES[c["dtype"]]
    rn = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=torch.float32).to(dt)  # noqa: E731
    if c["fused"]:
        q, k, v = rn(T, (NQ + 2 * NK) * HD).view(T, NQ + 2 * NK, HD).split([NQ, NK, NK], 1)
    else:
        q, k, v = rn(T, NQ, HD), rn(T, NK, HD), rn(T, NK, HD)
    # text advances all axes together, an image's tokens differ in their rows and columns
    step = torch.arange(T, device=dev) % max(1, c["far"] - 64)
    pos = torch.stack([step] + [step // 16 + torch.randint(0, 64, (T,), generator=g, device=dev) for _ in range(c["axes"] - 1)])
    s = {"q": q, "k": k, "v": v, "pos": pos.to(torch.int32), "axis": torch.tensor(_axis_of(c), device=dev),
         "freq": THETA ** (-torch.arange(0, HD, 2, dtype=torch.float64, device=dev) / HD), "wq": None, "wk": None}
    if c["norm"]:
        s["wq"], s["wk"] = (0.1 * rn(HD)).to(dt), (0.1 * rn(HD)).to(dt)
    if c["store"]:
        n_pages = _cdiv(T, c["P"]) + 3
        s["kp"], s["vp"] = rn(n_pages + 1, c["P"], NK, HD), rn(n_pages + 1, c["P"], NK, HD)  # one page more than is used
        slots = torch.randperm(n_pages * c["P"], generator=g, device=dev)[:T]
        s["slots"] = torch.where(torch.arange(T, device=dev) % 16 == 15, -1, slots)
        s["n_pages"] = n_pages
    if own:
        s["rope"] = _paged().AxesRotary(HD, _axis_of(c), theta=THETA, q_norm=s["wq"], k_norm=s["wk"], eps=EPS, device=dev)
    return s


def _prepare_attend(c, seed, dev, g):
    add, old, _ = _lens(c, seed)
    B, P, NQ, NK, HD, dt = c["B"], c["P"], c["NQ"], c["NK"], c["HD"], DTYPES[c["dtype"]]
    rn = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=dt)  # noqa: E731
    n = [a + o for a, o in zip(add, old)]
    held = [_cdiv(x, P) for x in n]
    T, n_pages = sum(add), sum(held) + 5
    perm = torch.randperm(n_pages, generator=g, device=dev, dtype=torch.int32)
    table = torch.full((B, max(held)), -1, dtype=torch.int32, device=dev)
    table[torch.arange(max(held), device=dev)[None, :] < torch.tensor(held, device=dev)[:, None]] = perm[: sum(held)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    cu = [0]
    for a in add:
        cu.append(cu[-1] + a)
    return {"q": rn(T + c["spare"], NQ, HD) * 2, "kp": rn(n_pages, P, NK, HD), "vp": rn(n_pages, P, NK, HD), "table": table,
            "cu": i32(cu), "kv_len": i32(n), "max_q": max(add), "max_kv": max(n), "out": torch.zeros(T + c["spare"], NQ, HD, dtype=dt, device=dev),
            "scale": HD ** -0.5, "causal": c["causal"], "window": c["window"], "sinks": c["sinks"], "case": c}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"map": _prepare_map, "rope": _prepare_rope, "attend": _prepare_attend}[case["op"]](case, seed, dev, g)
    s["op"] = case["op"]
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _map_plain(s):
    P, T, dev = s["P"], s["T"], s["add"].device
    n_pages, (B, cols) = s["queue"].numel(), s["table"].shape
    old, head, free = s["len"].long(), s["ends"][0].long(), s["ends"][1].long()
    done = s["done"] != 0 if s["done"] is not None else torch.zeros(B, dtype=torch.bool, device=dev)
    add = torch.where(done, 0, s["add"].clamp(min=0).long())
    held = (old + P - 1) // P
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), add.cumsum(0)])
    fits = ((old + add + P - 1) // P <= cols) & (cu[1:] <= T)
    need = torch.where(fits, (old + add + P - 1) // P - held, 0)
    last = need.cumsum(0)
    granted = fits & ((need == 0) | (last <= free)) & ~done
    first, need = last - need, torch.where(granted, need, 0)
    # the tokens: their request, their place in it, their page (an old one or one off the queue), their slot
    t = torch.arange(T, device=dev)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(0, B - 1)
    inside = t < cu[-1]
    pos = t - cu[b] + old[b]
    page = pos // P
    fresh = page - held[b]
    popped = s["queue"][(head + first[b] + fresh.clamp(min=0)) % n_pages]
    ok = inside & granted[b]
    at = torch.where(fresh >= 0, popped, s["table"][b, page.clamp(0, cols - 1)]).long()
    slots = torch.where(ok, at * P + pos % P, -1)
    # the table's new entries
    col = torch.arange(cols, device=dev)[None, :]
    new = (col >= held[:, None]) & (col < (held + need)[:, None])
    table = torch.where(new, s["queue"][(head + first[:, None] + (col - held[:, None]).clamp(min=0)) % n_pages], s["table"])
    # the ended requests' pages go to the queue's end
    back = torch.where(done, held, 0)
    put = (col < back[:, None])
    place = (head + free + (back.cumsum(0) - back)[:, None] + col) % n_pages
    queue = torch.cat([s["queue"], s["queue"][:1]])
    queue[torch.where(put, place, n_pages)] = torch.where(put, s["table"], queue[n_pages])
    took, gave = need.sum(), back.sum()
    kv_len = torch.where(done, 0, old + torch.where(granted, add, 0))
    return {"cu": cu.to(torch.int32), "slots": slots, "pos": torch.where(inside, pos, 0).to(torch.int32), "granted": granted.to(torch.int32),
            "kv_len": kv_len.to(torch.int32), "table": table, "queue": queue[:n_pages],
            "ends": torch.stack([(head + took) % n_pages, free - took + gave]).to(torch.int32)}


def _turn(x, w, cos, sin):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w.float())
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _rope_plain(s):
    angle = s["pos"][s["axis"]].double().t() * s["freq"]  # [T, HD / 2]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _turn(s["q"], s["wq"], cos, sin).to(s["q"].dtype)
    k = _turn(s["k"], s["wk"], cos, sin).to(s["k"].dtype)
    if "slots" not in s:
        return {"q": q, "k": k}
    N, P = s["n_pages"], s["kp"].shape[1]
    at = torch.where(s["slots"] >= 0, s["slots"], N * P)  # padding goes to the page that nobody uses
    s["kp"].view(-1, *k.shape[1:])[at] = k
    s["vp"].view(-1, *k.shape[1:])[at] = s["v"]
    return {"q": q, "k_pages": s["kp"][:N], "v_pages": s["vp"][:N]}


def _attend_plain(s):
    q, cu, n, P = s["q"], s["cu"].long(), s["kv_len"].long(), s["kp"].shape[1]
    (T, NQ, HD), NK, B, dev = q.shape, s["kp"].shape[2], n.shape[0], q.device
    Q, K, G = s["max_q"], s["max_kv"], NQ // s["kp"].shape[2]
    j, i = torch.arange(K, device=dev), torch.arange(Q, device=dev)
    # the requests side by side, padded to the longest: q [B, NK, G Q, HD], k and v [B, NK, K, HD]
    row = (cu[:-1, None] + i).clamp(max=T - 1)
    x = q[row].float().view(B, Q, NK, G, HD).permute(0, 2, 3, 1, 4).reshape(B, NK, G * Q, HD)
    page = s["table"].long().clamp(min=0)[:, j // P]
    here = (j < n[:, None])[:, :, None, None]
    k = torch.where(here, s["kp"][page, j % P], 0).float().transpose(1, 2).contiguous()
    v = torch.where(here, s["vp"][page, j % P], 0).float().transpose(1, 2).contiguous()
    p = (n - cu[1:] + cu[:-1])[:, None] + i  # the queries' positions
    see = (j < n[:, None])[:, None, :].expand(B, Q, K)
    if s["causal"]:
        see = see & (j <= p[:, :, None])
        if s["window"]:
            see = see & ((p[:, :, None] - j < s["window"]) | (j < s["sinks"]))
    score = torch.matmul(x, k.transpose(-1, -2).contiguous()).mul_(s["scale"]).view(B, NK, G, Q, K)
    score.masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(torch.isfinite(top), top, 0)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(B, NK, G * Q, K), v).view(B, NK, G, Q, HD) / torch.where(total > 0, total, 1)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Q, NQ, HD).to(q.dtype)
    t = torch.arange(T, device=dev)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(0, B - 1)
    s["out"].copy_(torch.where((t < cu[-1])[:, None, None], o[b, (t - cu[b]).clamp(0, Q - 1)], s["out"]))
    return s["out"]


def run(s):
    if own:
        if s["op"] == "map":
            m = s["pool"].map(s["add"], s["done"])
            return {"cu": m.cu, "slots": m.slots, "pos": m.pos, "granted": m.granted, "kv_len": m.kv_len, "table": m.table,
                    "queue": m.queue, "ends": m.ends}
        if s["op"] == "rope":
            if "slots" not in s:
                q, k = s["rope"](s["q"], s["k"], s["pos"])
                return {"q": q, "k": k}
            N = s["n_pages"]
            kp, vp = s["kp"][:N], s["vp"][:N]
            return {"q": s["rope"].store(s["q"], s["k"], s["v"], s["pos"], kp, vp, s["slots"]), "k_pages": kp, "v_pages": vp}
        return _paged().page_attend(s["q"], s["kp"], s["vp"], s["table"], s["cu"], s["kv_len"], max_q=s["max_q"], scale=s["scale"],
                                    causal=s["causal"], window=s["window"], sinks=s["sinks"], out=s["out"])
    return {"map": _map_plain, "rope": _rope_plain, "attend": _attend_plain}[s["op"]](s)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def _exact_rope(c, s):
    turns = {}
    for name, w in (("q", s["wq"]), ("k", s["wk"])):
        x = s[name].double()
        if w is not None:
            x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / c["HD"] + EPS) * (1 + w.double())
        z = torch.complex(x[..., : c["HD"] // 2], x[..., c["HD"] // 2:])  # a pair is a number of the plane, turned by its angle
        a = torch.stack([s["pos"][ax].double() * s["freq"][i] for i, ax in enumerate(_axis_of(c))], -1)
        z = z * torch.polar(torch.ones_like(a), a)[:, None]
        turns[name] = torch.cat([z.real, z.imag], -1)
    if not c["store"]:
        return turns
    N = s["n_pages"]
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    kp, vp = s["kp"][:N].double().flatten(0, 1), s["vp"][:N].double().flatten(0, 1)
    kp[at], vp[at] = turns["k"][keep], s["v"].double()[keep]
    return {"q": turns["q"], "k_pages": kp.view(N, c["P"], c["NK"], c["HD"]), "v_pages": vp.view(N, c["P"], c["NK"], c["HD"])}


def _exact_attend(c, s):
    out = s["out"].double()
    cu, G, P = s["cu"].tolist(), c["NQ"] // c["NK"], c["P"]
    for b, n in enumerate(s["kv_len"].tolist()):
        nq = cu[b + 1] - cu[b]
        pages = s["table"][b, : _cdiv(n, P)].long()
        k, v = (s[x][pages].flatten(0, 1)[:n].double() for x in ("kp", "vp"))
        for lo in range(0, nq, 1024):
            hi = min(nq, lo + 1024)
            p = torch.arange(n - nq + lo, n - nq + hi, device=k.device)[:, None]
            j = torch.arange(n, device=k.device)[None, :]
            hide = torch.zeros(hi - lo, n, dtype=torch.bool, device=k.device)
            if c["causal"]:
                hide |= j > p
                if c["window"]:
                    hide |= (p - j >= c["window"]) & (j >= c["sinks"])
            for h in range(c["NQ"]):
                x = s["q"][cu[b] + lo: cu[b] + hi, h].double() @ k[:, h // G].t().contiguous() * s["scale"]
                x = x.masked_fill(hide, -math.inf)
                out[cu[b] + lo: cu[b] + hi, h] = torch.exp(x - torch.logsumexp(x, -1, keepdim=True)) @ v[:, h // G].contiguous()
    return out


def exact(case, seed):
    if case["op"] == "map":
        return None  # whole numbers
    if case["op"] == "attend" and case["B"] * case["NQ"] * _cdiv(case["hi"], 1024) > 20000:
        return None
    s = prepare(case, seed)
    return _exact_rope(case, s) if case["op"] == "rope" else _exact_attend(case, s)
