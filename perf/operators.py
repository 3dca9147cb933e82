"""Cases that measure the decode loop's key/value cache operators: storing new tokens in a cache that is quantised as it
is written and reading rows back, attention with a sliding window and always-visible first tokens over that cache, and
attention of a tree of drafted tokens over it with the move of the accepted path.

`run` computes each pass in its plain form (elementary torch operations in 32 bits, one rounding at the end), or, where
`own` is set, through nwc_b200.KVCache.  `exact` gives the same results from the definitions in 64 bits.

Definitions.  A cache holds, per key/value head, `capacity` slots of head_dim numbers for K and for V.  Position p lives in
slot p, or, with a window, in slot p for p < sinks and sinks + (p - sinks) mod (capacity - sinks) otherwise.  bf16 caches
hold the value rounded to bf16; fp8 caches hold e4m3 codes and per row one byte b: value = code * 2^(b - 127), with the
smallest exponent for which the row's largest magnitude is at most 448 * 2^(b - 127).
"""
import math

import torch

own = False

EPS = 1e-6
THETA = 1e6


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of the decode loop enters the cache (Qwen3-0.6B heads): launch latency
        dict(name="store one token fp8", op="store", elem="fp8", n_q=16, n_kv=8, hd=128, T=1, pos=777, capacity=1024, window=0, sinks=0, norm=True),
        # a chunk of a prompt wraps around a ring of a window of 1000 (Qwen3-4B heads)
        dict(name="store 517 tokens fp8 ring", op="store", elem="fp8", n_q=32, n_kv=8, hd=128, T=517, pos=2900, capacity=1600, window=1000, sinks=4, norm=True),
        # a long prompt chunk (Llama-3-70B heads): bandwidth
        dict(name="store 4096 tokens fp8", op="store", elem="fp8", n_q=64, n_kv=8, hd=128, T=4096, pos=4096, capacity=8192, window=0, sinks=0, norm=False),
        # a session's whole cache of one layer read back as bf16
        dict(name="read 60001 tokens fp8", op="read", elem="fp8", n_q=8, n_kv=8, hd=128, T=60001, pos=17, capacity=65536, window=0, sinks=0, norm=False),
        # a decode step of a streaming session: window of 1024 plus four first tokens, far beyond the ring's length
        dict(name="one token window 1024 fp8", op="window", elem="fp8", n_q=16, n_kv=8, hd=128, T=1, pos=5000, capacity=1100, window=1024, sinks=4, norm=True),
        # a decode step over a full bf16 cache of ordinary length
        dict(name="one token over 8191 bf16", op="window", elem="bf16", n_q=32, n_kv=8, hd=128, T=1, pos=8190, capacity=8192, window=0, sinks=0, norm=True),
        # a decode step over a very long quantised cache: bandwidth
        dict(name="one token over 131071 fp8", op="window", elem="fp8", n_q=64, n_kv=8, hd=128, T=1, pos=131070, capacity=131072, window=0, sinks=0, norm=False),
        # a prompt chunk under a sliding window: matrix products
        dict(name="4096 tokens window 4096 bf16", op="window", elem="bf16", n_q=32, n_kv=8, hd=128, T=4096, pos=8192, capacity=16384, window=4096, sinks=4, norm=True),
        # an odd prompt chunk behind a long quantised context, everything visible
        dict(name="1000 tokens over 24000 fp8", op="window", elem="fp8", n_q=64, n_kv=8, hd=128, T=1000, pos=23999, capacity=25000, window=0, sinks=0, norm=False),
        # a small draft tree over a short conversation
        dict(name="tree of 26 over 700 bf16", op="tree", elem="bf16", n_q=16, n_kv=8, hd=128, T=26, pos=700, capacity=1024, window=0, sinks=0, norm=True),
        # a large draft tree over a long quantised context
        dict(name="tree of 64 over 32768 fp8", op="tree", elem="fp8", n_q=64, n_kv=8, hd=128, T=64, pos=32768, capacity=33000, window=0, sinks=0, norm=False),
        # a whole verification: the tree enters the ring, attends, and the accepted path is moved together
        dict(name="verify tree of 48 fp8 ring", op="verify", elem="fp8", n_q=32, n_kv=8, hd=128, T=48, pos=9001, capacity=2200, window=2048, sinks=4, norm=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["store", "read", "window", "window", "tree", "verify"])
        n_q, n_kv, hd = rng.choice([(16, 8, 128), (32, 8, 128), (64, 8, 128), (4, 2, 64), (8, 1, 128), (6, 2, 128), (5, 5, 64), (8, 2, 256)])
        T = {"store": _spread(rng, 1, 4096), "read": _spread(rng, 1, 60001), "window": 1 if rng.random() < 0.4 else _spread(rng, 2, 4096),
             "tree": rng.randint(2, 64), "verify": rng.randint(2, 64)}[op]
        pos = _spread(rng, 1, 131070 if T == 1 else 32768)
        window, sinks = 0, 0
        if op != "read" and rng.random() < 0.5: window, sinks = _spread(rng, 16, 4096), rng.choice([0, 1, 4, 7])
        capacity = sinks + window + T + rng.randint(0, 100) if window else pos + T + rng.randint(0, 100)
        case = dict(op=op, elem=rng.choice(["bf16", "fp8"]), n_q=n_q, n_kv=n_kv, hd=hd, T=T, pos=pos, capacity=capacity, window=window, sinks=sinks,
                    norm=rng.random() < 0.5)
        w = work(case)
        seen = (min(pos, window + sinks) if window else pos) + T
        if w["flops"] <= 8.0e11 and w["bytes"] <= 3.0e8 and n_q * T * seen <= 1.6e9 or op in ("store", "read") and w["bytes"] <= 3.0e8: return case


# ---- inputs --------------------------------------------------------------------------------------------------------

def _slots(p, case):
    if not case["window"]: return p
    ring = case["capacity"] - case["sinks"]
    return torch.where(p < case["sinks"], p, case["sinks"] + (p - case["sinks"]) % ring)


def _power(e):
    """2^e in 32 bits for -127 <= e <= 127, from its bits: a power function need not be exact."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _quantise(x):
    """Rows of fp32 numbers -> e4m3 codes and the exponent byte of each row."""
    m, e = torch.frexp(x.abs().amax(-1))                             # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875)
    b = torch.where(m == 0, torch.zeros_like(e), (e + 127).clamp(0, 254))
    return (x * _power(127 - b)[..., None]).to(torch.float8_e4m3fn), b.to(torch.uint8)


def _values(codes, byte):
    return codes.float() * _power(byte.int() - 127)[..., None]


def _draft_tree(T, gen):
    """Parents of a draft tree in the order a drafter proposes it: a node hangs below one of the last dozen."""
    parents = [-1]
    for i in range(1, T): parents.append(int(torch.randint(max(0, i - 12), i, (1,), generator=gen)))
    depth, seen = [0] * T, [[0] * ((T + 31) // 32) for _ in range(T)]
    for i, p in enumerate(parents):
        if p >= 0: depth[i] = depth[p] + 1; seen[i] = list(seen[p])
        seen[i][i // 32] |= 1 << (i % 32)
    path, at = [], max(range(T), key=lambda i: (depth[i], i))         # the accepted path: root to the deepest node
    while at >= 0: path.insert(0, at); at = parents[at]
    signed = [[w - (1 << 32) if w >= 1 << 31 else w for w in row] for row in seen]
    return torch.tensor(depth, dtype=torch.int32), torch.tensor(signed, dtype=torch.int32), torch.tensor(path, dtype=torch.int32)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    n_q, n_kv, hd, T, cap, pos = (case[k] for k in ("n_q", "n_kv", "hd", "T", "capacity", "pos"))
    s = {"case": case, "pos": torch.tensor([pos], dtype=torch.int32, device=dev)}
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev)
    # cached keys and values: normal, every channel with its own spread, as projections give them
    spread = lambda: torch.exp(0.3 * randn(n_kv, 1, hd))
    for name in ("k", "v"):
        x = (randn(n_kv, cap, hd) * spread()).to(torch.bfloat16)
        s[name + "_exp"] = None
        if case["elem"] == "fp8":
            x, b = _quantise(x.float())
            s[name + "_exp"] = b[None].contiguous()
        s[name] = x[None].contiguous()                                # [layers = 1][n_kv][capacity][hd]
    if case["op"] in ("store", "verify"):
        s["qkv"] = (1.5 * randn(T, (n_q + 2 * n_kv) * hd)).to(torch.bfloat16)
        s["q_norm"] = (1 + 0.2 * randn(hd)).to(torch.bfloat16) if case["norm"] else None
        s["k_norm"] = (1 + 0.2 * randn(hd)).to(torch.bfloat16) if case["norm"] else None
        angle = torch.arange(pos + T, dtype=torch.float64, device=dev)[:, None] * THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=dev) / hd)
        angle = torch.cat([angle, angle], -1)
        s["cos"], s["sin"] = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    elif case["op"] != "read":
        s["q"] = (2.0 * randn(T, n_q, hd)).to(torch.bfloat16)
    s["depth"] = s["visible"] = None
    if case["op"] in ("tree", "verify"):
        depth, visible, path = _draft_tree(T, torch.Generator().manual_seed(seed))
        s["depth"], s["visible"], s["path"] = depth.to(dev), visible.to(dev), path.to(dev)
        s["accepted"] = torch.tensor([path.numel()], dtype=torch.int32, device=dev)
        s["n_accepted"] = path.numel()
    if own:                                                          # the handle a program keeps: it refers to the tensors above
        from nwc_b200 import KVCache
        s["cache"] = KVCache.over(s["k"], s["v"], s["k_exp"], s["v_exp"], window=case["window"], sinks=case["sinks"])
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    case, cache = s["case"], s["cache"]
    op, pos = case["op"], s["pos"]
    if op == "store":
        q = cache.append(s["qkv"], pos, s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        k, v = cache.read(case["pos"], case["T"])
        return {"q": q, "k": k, "v": v}
    if op == "read":
        k, v = cache.read(case["pos"], case["T"])
        return {"k": k, "v": v}
    if op == "window": return {"out": cache.attend(s["q"], pos)}
    if op == "tree": return {"out": cache.attend(s["q"], pos, visible=s["visible"], depth=s["depth"])}
    q = cache.append(s["qkv"], pos, s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, depth=s["depth"])
    out = cache.attend(q, pos, visible=s["visible"], depth=s["depth"])
    cache.commit(pos, s["path"], s["accepted"])
    k, v = cache.read(case["pos"], case["T"])
    return {"out": out, "k": k, "v": v}


def _run_plain(s):
    case = s["case"]
    op, T, pos, hd = case["op"], case["T"], case["pos"], case["hd"]
    new = torch.arange(pos, pos + T, device=s["k"].device)
    if op == "read":
        k, v = _plain_rows(s, _slots(new, case))
        return {"k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)}
    if op == "window": return {"out": _plain_attend(s, s["q"].float())}
    if op == "tree": return {"out": _plain_attend(s, s["q"].float())}
    q = _plain_store(s, new)
    if op == "store":
        k, v = _plain_rows(s, _slots(new, case))
        return {"q": q, "k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)}
    out = _plain_attend(s, q.float())
    n = s["n_accepted"]
    _plain_move(s, _slots(pos + s["path"][:n].long(), case), _slots(new[:n], case))
    k, v = _plain_rows(s, _slots(new, case))
    return {"out": out, "k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)}


def _plain_rows(s, slots):
    """K and V of the given slots in 32 bits, [n_kv][slots][hd]."""
    if s["k_exp"] is None: return s["k"][0][:, slots].float(), s["v"][0][:, slots].float()
    byte = lambda name: s[name + "_exp"][0][:, slots]
    codes = lambda name: s[name][0].view(torch.uint8)[:, slots].view(torch.float8_e4m3fn)
    return _values(codes("k"), byte("k")), _values(codes("v"), byte("v"))


def _plain_store(s, new):
    case = s["case"]
    n_q, n_kv, hd, T = case["n_q"], case["n_kv"], case["hd"], case["T"]
    x = s["qkv"].float().view(T, n_q + 2 * n_kv, hd)
    q, k, v = x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
    if s["q_norm"] is not None:
        q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"].float()
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"].float()
    at = new if s["depth"] is None else new[0] + s["depth"].long()
    c, sn = s["cos"].float()[at][:, None], s["sin"].float()[at][:, None]
    turn = lambda t: t * c + torch.cat([-t[..., hd // 2:], t[..., :hd // 2]], -1) * sn
    q, k = turn(q), turn(k)
    slots = _slots(new, case)
    k, v = k.transpose(0, 1), v.transpose(0, 1)
    if s["k_exp"] is None:
        s["k"][0][:, slots], s["v"][0][:, slots] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    else:
        (kc, kb), (vc, vb) = _quantise(k), _quantise(v)
        s["k"][0].view(torch.uint8)[:, slots], s["v"][0].view(torch.uint8)[:, slots] = kc.view(torch.uint8), vc.view(torch.uint8)
        s["k_exp"][0][:, slots], s["v_exp"][0][:, slots] = kb, vb
    return q.to(torch.bfloat16)


def _plain_move(s, source, target):
    raw = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    rows = lambda t: raw(t)[0][:, source].clone()
    if s["k_exp"] is not None: s["k_exp"][0][:, target], s["v_exp"][0][:, target] = rows(s["k_exp"]), rows(s["v_exp"])
    raw(s["k"])[0][:, target], raw(s["v"])[0][:, target] = rows(s["k"]), rows(s["v"])


def _plain_attend(s, q):
    case = s["case"]
    n_q, n_kv, hd, T, pos, window, sinks = (case[k] for k in ("n_q", "n_kv", "hd", "T", "pos", "window", "sinks"))
    dev = q.device
    first = max(0, pos + 1 - window) if window else 0
    at = torch.cat([torch.arange(min(sinks, first), device=dev), torch.arange(first, pos + T, device=dev)])
    k, v = _plain_rows(s, _slots(at, case))
    t = torch.arange(T, device=dev)
    mine = pos + (t if s["depth"] is None else s["depth"].long())[:, None]
    sees = (at < sinks) | (at > mine - window) if window else torch.ones(T, at.numel(), dtype=torch.bool, device=dev)
    if s["visible"] is None: sees = sees & (at <= mine)
    else:
        j = (at - pos).clamp(0, T - 1)
        bit = (s["visible"][:, j // 32] >> (j % 32)) & 1
        sees = torch.where(at < pos, sees, bit.bool())
    rows = q.view(T, n_kv, n_q // n_kv, hd).permute(1, 2, 0, 3).reshape(n_kv, -1, hd)
    x = (rows @ k.transpose(1, 2)).view(n_kv, n_q // n_kv, T, -1) / math.sqrt(hd)
    x = x.masked_fill(~sees, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    total = x.sum(-1, keepdim=True)
    o = (x.view(n_kv, -1, at.numel()) @ v).view(n_kv, n_q // n_kv, T, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(2, 0, 1, 3).reshape(T, n_q * hd).to(torch.bfloat16)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    op, n_q, n_kv, hd, T, pos, window, sinks = (case[k] for k in ("op", "n_q", "n_kv", "hd", "T", "pos", "window", "sinks"))
    row = hd + 1 if case["elem"] == "fp8" else 2 * hd                 # bytes of one cached row of one head
    if op == "read": return {"bytes": T * n_kv * 2 * (row + 2 * hd), "flops": 0}
    store = T * ((n_q + 2 * n_kv) * hd * 2 + 4 * hd + n_q * hd * 2 + 2 * n_kv * row)
    if op == "store": return {"bytes": store + T * n_kv * 2 * 2 * hd, "flops": 0}
    # cached rows that some token sees, and pairs of a token and a row it sees (of a tree: its ancestors count as half of it)
    first = max(0, pos + 1 - window) if window else 0
    rows = pos + T - first + min(sinks, first)
    if op == "window":
        pairs = 0
        if window:
            full = max(0, min(T, window - 1 - pos))                   # tokens whose window reaches below position 0
            pairs += full * (pos + 1) + full * (full - 1) // 2 + (T - full) * window
            for t in range(full, T):
                missing = min(sinks, pos + t + 1 - window)
                if missing == sinks: pairs += (T - t) * sinks; break
                pairs += missing
        else: pairs = T * (pos + 1) + T * (T - 1) // 2
    else:
        pairs = T * (rows - T) + T * (T + 1) // 2
    attend = {"bytes": rows * n_kv * 2 * row + 2 * T * n_q * hd * 2, "flops": 4 * hd * n_q * pairs}
    if op == "verify": attend["bytes"] += store - T * 2 * n_kv * row - T * n_q * hd * 2      # the stored rows and q are counted once
    return attend


# ---- the same results from the definitions, in 64 bits --------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    n_q, n_kv, hd, T, pos, window, sinks = (case[k] for k in ("n_q", "n_kv", "hd", "T", "pos", "window", "sinks"))
    ring = case["capacity"] - sinks
    two_to = lambda e: ((e.long() + 1023) << 52).view(torch.float64)
    slot = lambda p: p if not window or p < sinks else sinks + (p - sinks) % ring
    held = {}
    for name in ("k", "v"):
        held[name] = s[name][0].to(torch.float64)
        if s[name + "_exp"] is not None: held[name] = held[name] * two_to(s[name + "_exp"][0].long() - 127)[..., None]
    fresh = torch.tensor([slot(pos + t) for t in range(T)], device="cuda")
    q = s["q"].double() if "q" in s else None
    if case["op"] == "read": return {"k": held["k"].index_select(1, fresh), "v": held["v"].index_select(1, fresh)}
    if case["op"] in ("store", "verify"):
        parts = s["qkv"].double().split([n_q * hd, n_kv * hd, n_kv * hd], 1)
        q, k, v = (p.reshape(T, -1, hd) for p in parts)
        where = pos + (s["depth"].long() if s["depth"] is not None else torch.arange(T, device="cuda"))
        cos, sin = s["cos"][where].double().unsqueeze(1), s["sin"][where].double().unsqueeze(1)
        h = hd // 2
        def turned(x, weight):
            if weight is not None: x = x * (x.pow(2).sum(-1, keepdim=True) / hd + EPS).pow(-0.5) * weight.double()
            lo, hi = x[..., :h], x[..., h:]
            return torch.cat([lo * cos[..., :h] - hi * sin[..., :h], hi * cos[..., h:] + lo * sin[..., h:]], -1)
        q, k = turned(q, s["q_norm"]), turned(k, s["k_norm"])
        def as_held(x):
            if case["elem"] == "bf16": return x.to(torch.bfloat16).double()
            top = x.abs().amax(-1, keepdim=True)
            unit = two_to(torch.ceil(torch.log2(top / 448)))
            unit = torch.where(top > 448 * unit, 2 * unit, torch.where(top <= 224 * unit, unit / 2, unit))
            y = x / unit
            step = two_to(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
            return torch.round(y / step) * step * unit
        rows = {"k": as_held(k), "v": as_held(v)}
        for name in ("k", "v"): held[name].index_copy_(1, fresh, rows[name].transpose(0, 1).contiguous())
        if case["op"] == "store": return {"q": q, "k": rows["k"].transpose(0, 1), "v": rows["v"].transpose(0, 1)}
        q = q.to(torch.bfloat16).double()                             # the attention reads what the store wrote
    t = torch.arange(T, device="cuda").unsqueeze(1)
    out = torch.zeros(T, n_q, hd, dtype=torch.float64, device="cuda")
    low = max(0, pos + 1 - window) if window else 0
    logical = list(range(min(sinks, low))) + list(range(low, pos + T))
    key_pos = torch.tensor(logical, device="cuda").unsqueeze(0)
    key_slot = torch.tensor([slot(p) for p in logical], device="cuda")
    if s["visible"] is None:
        mask = key_pos <= pos + t
        if window: mask &= (key_pos < sinks) | (pos + t - key_pos < window)
    else:
        mask = key_pos < pos
        if window: mask = mask & ((key_pos < sinks) | (pos + s["depth"].long().unsqueeze(1) - key_pos < window))
        words = s["visible"].long() & 0xFFFFFFFF
        drafted = torch.stack([(words[:, j // 32] >> (j % 32)) & 1 for j in range(T)], 1).bool()
        mask = torch.cat([mask.expand(T, -1)[:, :len(logical) - T], drafted], 1)
    for h in range(n_q):
        kv = h * n_kv // n_q
        w = q[:, h] @ held["k"][kv].index_select(0, key_slot).T * hd ** -0.5
        w = torch.where(mask, w, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
        out[:, h] = torch.nan_to_num(torch.softmax(w, -1)) @ held["v"][kv].index_select(0, key_slot)
    out = out.reshape(T, n_q * hd)
    if case["op"] != "verify": return {"out": out}
    way = [int(i) for i in s["path"]]                                 # the accepted rows first; those behind them stay as they were stored
    way += list(range(len(way), T))
    return {"out": out, "k": rows["k"][way].transpose(0, 1), "v": rows["v"][way].transpose(0, 1)}
