"""Cases that measure the operators around the paged key-value cache: attention of one new token, attention of a
prompt with a sliding window and leading tokens that stay visible, the weight that each cached token has received,
and eviction from the cache by that weight.

A cached token n is visible to a query at position p iff n <= p and (window == 0 or n > p - window or n < sinks);
query row r of a sequence with q_len rows and kv_len cached tokens has position kv_len - q_len + r.  With `own` the
calls go to swiftlm_b200.kernels; without it the same values are computed by elementary torch operations in 32 bits.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one sequence in a chat, the shortest call: latency
        dict(name="decode one short", op="decode", B=1, Hq=16, Hkv=2, D=256, dtype="bf16", page=0, N=517, ragged=False, window=0, sinks=0, mass=False, lse=False),
        # a serving batch at the benchmark's head layout, lengths of their own, and a cache that will be evicted from
        dict(name="decode batch with weights", op="decode", B=32, Hq=16, Hkv=2, D=256, dtype="bf16", page=256, N=8208, ragged=True, window=0, sinks=0, mass=True, lse=True),
        # the benchmark's long contexts behind its page table
        dict(name="decode long", op="decode", B=8, Hq=16, Hkv=2, D=256, dtype="bf16", page=256, N=102400, ragged=True, window=0, sinks=0, mass=False, lse=False),
        # the draft model's sink and window over a long cache, small pages
        dict(name="decode window", op="decode", B=64, Hq=32, Hkv=8, D=128, dtype="f16", page=64, N=16384, ragged=True, window=1024, sinks=64, mass=False, lse=True),
        # a few short prompts of unequal length in small pages
        dict(name="prompt short ragged", op="prompt", B=5, Hq=12, Hkv=4, D=64, dtype="f16", page=16, T=193, N=331, ragged=True, window=0, sinks=0, lse=True),
        # one chunk of a long prompt over what earlier chunks left in the cache (chunks of 2048 tokens)
        dict(name="prompt chunk", op="prompt", B=1, Hq=16, Hkv=2, D=256, dtype="bf16", page=256, T=2048, N=10240, ragged=False, window=0, sinks=0, lse=False),
        # the draft model's sink and window over a whole prompt
        dict(name="prompt window", op="prompt", B=2, Hq=32, Hkv=8, D=128, dtype="bf16", page=0, T=8192, N=8192, ragged=False, window=1024, sinks=64, lse=True),
        # a whole prompt at once: the largest
        dict(name="prompt whole", op="prompt", B=1, Hq=16, Hkv=2, D=256, dtype="bf16", page=0, T=8192, N=8192, ragged=False, window=0, sinks=0, lse=True),
        # the weights that a verify block of 16 rows gave to a batch's caches
        dict(name="mass of a block", op="mass", B=32, Hq=16, Hkv=2, D=256, dtype="bf16", page=256, T=16, N=4112, ragged=True, window=0, sinks=0),
        # the weights of a prompt chunk over the whole cache, before the cache is cut to its budget
        dict(name="mass of a chunk", op="mass", B=1, Hq=32, Hkv=8, D=128, dtype="bf16", page=0, T=2048, N=16384, ragged=False, window=0, sinks=0),
        # a cache at its budget that has just taken a block of 16: back to 64 sinks and 1024 tokens
        dict(name="evict a block", op="evict", B=32, Hkv=2, D=256, dtype="bf16", page=128, N=1104, ragged=False, budget=1088, recent=512, sinks=64),
        # long prompts cut down to a budget
        dict(name="evict a prompt", op="evict", B=8, Hkv=2, D=256, dtype="bf16", page=256, N=32768, ragged=True, budget=4096, recent=1024, sinks=64),
    ]


MOST_FLOPS, MOST_BYTES = 5.4e11, 1.6e9      # no drawn case is larger than the largest listed ones


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = dict(op=rng.choice(["decode", "decode", "prompt", "prompt", "mass", "evict"]))
        Hkv = rng.choice([1, 2, 3, 4, 8])
        G = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        c.update(B=_log(rng, 1, 64), Hq=Hkv * G, Hkv=Hkv, D=rng.choice([64, 128, 256]), dtype=rng.choice(["bf16", "f16"]),
                 page=rng.choice([0, 0, 16, 48, 64, 128, 256]), ragged=rng.random() < 0.6)
        window = rng.choice([0, 0, 1]) and _log(rng, 1, 4096)
        sinks = rng.choice([0, 4, 64, _log(rng, 1, 200)]) if window else 0
        if c["op"] == "decode":
            c.update(N=_log(rng, 1, 102400), window=window, sinks=sinks, mass=rng.random() < 0.4, lse=rng.random() < 0.5)
        elif c["op"] == "prompt":
            c.update(T=_log(rng, 1, 8192), window=window, sinks=sinks, lse=rng.random() < 0.5)
            c["N"] = c["T"] + rng.choice([0, 0, _log(rng, 1, 16384)])
        elif c["op"] == "mass":
            c.update(T=_log(rng, 1, 2048), window=window, sinks=sinks)
            c["N"] = c["T"] + rng.choice([0, _log(rng, 1, 32768)])
        else:
            c.pop("Hq")
            c["N"] = _log(rng, 2, 32768)
            c["budget"] = _log(rng, 1, c["N"])
            c["recent"] = rng.randint(0, c["budget"] // 2)
            c["sinks"] = rng.randint(0, min(64, c["budget"] - c["recent"]))
        w = work(c)
        rows = c["B"] * c.get("Hq", 1) * c.get("T", 1) * c["N"]
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and c["B"] * c["Hkv"] * c["N"] * c["D"] <= 4.5e8 and rows <= 1.1e9:
            return c


# ---- lengths: a part of the case, not of the seed, because the work goes by them ----
def _spread(c, b, lo, hi):
    return hi if not c["ragged"] else max(lo, hi - int((hi - lo) * ((b * 0.6180339887498949 + 0.3) % 1.0)))


def _lengths(c):
    """(kv_len, q_len) of each sequence.  Ragged: between a third of the longest and the longest."""
    kv, ql = [], []
    for b in range(c["B"]):
        t = _spread(c, b, (c.get("T", 1) + 2) // 3, c.get("T", 1))
        past = _spread(c, b + 1, (c["N"] - c.get("T", 1) + 2) // 3, c["N"] - c.get("T", 1))
        ql.append(t)
        kv.append(t + past)
    return kv, ql


def _visible(c):
    """(pairs of a query and a visible key, keys visible to some query), summed over the sequences."""
    pairs = keys = 0
    for n, t in zip(*_lengths(c)):
        p = torch.arange(n - t, n, dtype=torch.float64)
        W, S = c["window"], c["sinks"]
        if W == 0:
            pairs += int((p + 1).sum())
            keys += n
        else:
            first = (p - W + 1).clamp(min=0)
            pairs += int((p + 1 - first + torch.minimum(first, torch.full_like(first, S))).sum())
            lo = max(0, n - t - W + 1)
            keys += n - lo + min(lo, S)
    return pairs, keys


def work(c):
    size = 2
    if c["op"] == "evict":
        nbytes = 0
        for n in _lengths(c)[0]:
            kept = min(n, c["budget"])
            moved = kept - min(kept, c["sinks"]) if n > kept else 0
            nbytes += c["Hkv"] * (4 * n + 8 * kept + moved * c["D"] * size * 4) + 8    # weights, places, rows read and written
        return {"bytes": nbytes, "flops": 0}
    pairs, keys = _visible(c)
    rows = sum(_lengths(c)[1]) * c["Hq"]
    kv = keys * c["Hkv"] * c["D"] * size
    if c["op"] == "mass":
        return {"bytes": kv + rows * (c["D"] * size + 4) + keys * c["Hkv"] * 8, "flops": 2 * pairs * c["Hq"] * c["D"]}
    nbytes = 2 * kv + 2 * rows * c["D"] * size + (rows * 4 if c["lse"] else 0) + (keys * c["Hkv"] * 8 if c.get("mass") else 0)
    return {"bytes": nbytes, "flops": 4 * pairs * c["Hq"] * c["D"]}


# ---- inputs ----
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32).to(dt)

    kv_len, q_len = (torch.tensor(x, dtype=torch.int32, device=dev) for x in _lengths(c))
    B, Hkv, D, N = c["B"], c["Hkv"], c["D"], c["N"]
    s = dict(c, kv_len=kv_len, q_len=q_len, scale=1.0 / math.sqrt(D), table=None)
    if c["page"]:
        pages = -(-N // c["page"])
        pool = B * pages + 3                                         # some pages of the pool belong to nobody
        s["table"] = torch.randperm(pool, device=dev, generator=g)[:B * pages].view(B, pages).to(torch.int32)
        shape, cap = (pool, Hkv, c["page"], D), pages * c["page"]
    else:
        shape, cap = (B, Hkv, N, D), N
    s["k"], s["v"] = normal(*shape), normal(*shape)
    if c["op"] == "evict" or c["op"] == "mass" or c.get("mass"):
        # accumulated weights are skewed: most tokens have little
        s["mass"] = torch.empty(B, Hkv, cap, device=dev).exponential_(generator=g).square_()
        s["mass"] *= torch.arange(cap, device=dev) < kv_len[:, None, None]
    if c["op"] == "evict":
        s["kept"] = torch.full((B, Hkv, c["budget"]), -1, dtype=torch.int32, device=dev)
        s["mass_out"] = torch.zeros_like(s["mass"])
        s["kv_len_out"] = torch.zeros_like(kv_len)
    elif c["op"] == "decode":
        s["q"] = normal(B, c["Hq"], D)
    else:
        s["q"] = normal(B, c["Hq"], c["T"], D)
        s["out"] = torch.zeros_like(s["q"])                          # rows behind a sequence's last query stay as they are
        if c["op"] == "mass":
            s["lse"] = _attend(s, s["q"], values=False)[1]
    return s


def _rows(pool, table):
    """[B, Hkv, capacity, D] of a page pool."""
    if table is None:
        return pool
    return pool[table.long()].transpose(1, 2).flatten(2, 3)


def _mask(s, T, cap):
    """[B, 1, 1, T, cap]: which key a query row sees; rows behind the last query see nothing."""
    r = torch.arange(T, device=s["kv_len"].device)
    n = torch.arange(cap, device=r.device)
    ql = s["q_len"][:, None]
    p = (s["kv_len"][:, None] - ql + r)[:, :, None]                   # [B, T, 1]
    seen = (n <= p) & (r < ql)[:, :, None]
    if s["window"]:
        seen &= (n > p - s["window"]) | (n < s["sinks"])
    return seen[:, None, None]


def _scores(s, q):
    k = _rows(s["k"], s["table"]).float()
    B, Hq, T, D = q.shape
    x = q.float().view(B, s["Hkv"], -1, T, D) @ k[:, :, None].transpose(-1, -2) * s["scale"]
    return x.masked_fill_(~_mask(s, T, k.shape[2]), -math.inf)


def _attend(s, q, values=True):
    """Plain form: (out, lse, weights) in 32 bits."""
    B, Hq, T, D = q.shape
    x = _scores(s, q)
    top = x.amax(-1, keepdim=True)
    p = (x - top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).view(B, Hq, T)
    p /= total.masked_fill(total == 0, 1.0)
    if not values:
        return None, lse, p
    o = p @ _rows(s["v"], s["table"]).float()[:, :, None]
    return o.view(B, Hq, T, D).to(q.dtype), lse, p


def _plain(s):
    if s["op"] == "decode":
        out, lse, p = _attend(s, s["q"][:, :, None])
        if s["mass"] is not False:
            s["mass"] += p.sum((2, 3))
        return [out[:, :, 0]] + ([lse[:, :, 0]] if s["lse"] else []) + ([s["mass"]] if s["mass"] is not False else [])
    if s["op"] == "prompt":
        out, lse, _ = _attend(s, s["q"])
        live = torch.arange(s["T"], device=out.device) < s["q_len"][:, None]
        s["out"].copy_(torch.where(live[:, None, :, None], out, s["out"]))
        return [s["out"]] + ([lse] if s["lse"] else [])
    if s["op"] == "mass":
        x, lse = _scores(s, s["q"]), s["lse"].view(s["B"], s["Hkv"], -1, s["T"], 1)
        s["mass"] += (x - lse.masked_fill(lse == -math.inf, 0.0)).exp_().sum((2, 3))
        return [s["mass"]]
    # eviction: the first `sinks`, the last `recent` and the heaviest of the others, in the order they are in
    cap, dev = s["mass"].shape[2], s["mass"].device
    n = torch.arange(cap, device=dev)
    length = s["kv_len"][:, None, None].long()
    left = length.clamp(max=s["budget"])
    keep = (n < s["sinks"]) | (n >= length - s["recent"])
    rank_of = torch.where(keep, math.inf, s["mass"]).masked_fill(n >= length, -math.inf)
    order = rank_of.sort(dim=-1, descending=True, stable=True).indices
    slot = torch.arange(s["budget"], device=dev).clamp(max=cap - 1)
    used = slot < left
    place = order[..., :s["budget"]] if cap >= s["budget"] else order[..., slot]
    kept = torch.where(used, place, cap).sort(dim=-1).values           # ascending; unused places last
    from_ = kept.clamp(max=cap - 1)
    b = torch.arange(s["B"], device=dev)[:, None, None].expand_as(from_)
    h = torch.arange(s["Hkv"], device=dev)[None, :, None].expand_as(from_)
    at = used.expand_as(from_).nonzero(as_tuple=True)
    bb, hh, src, dst = b[at], h[at], from_[at], at[2]
    for x in (s["k"], s["v"]):
        if s["table"] is None:
            x[bb, hh, dst] = x[bb, hh, src]
        else:
            t, pt = s["table"].long(), s["page"]
            x[t[bb, dst // pt], hh, dst % pt] = x[t[bb, src // pt], hh, src % pt]
    s["mass_out"].masked_fill_(n < length, 0.0)
    s["mass_out"][bb, hh, dst] = s["mass"][bb, hh, src]
    s["kept"].copy_(torch.where(used, kept, -1))
    s["kv_len_out"].copy_(left.view(-1))
    return [s["k"], s["v"], s["mass_out"], s["kept"], s["kv_len_out"]]


def run(state):
    s = state
    if not own:
        return _plain(s)
    from swiftlm_b200 import kernels
    if s["op"] == "decode":
        mass = None if s["mass"] is False else s["mass"]
        got = kernels.decode_sdpa(s["q"], s["k"], s["v"], s["scale"], kv_len=s["kv_len"], page_table=s["table"], window=s["window"],
                                  sinks=s["sinks"], mass=mass, return_lse=s["lse"], n_max=s["N"])
        return (list(got) if s["lse"] else [got]) + ([mass] if mass is not None else [])
    if s["op"] == "prompt":
        got = kernels.prompt_sdpa(s["q"], s["k"], s["v"], s["scale"], q_len=s["q_len"], kv_len=s["kv_len"], page_table=s["table"],
                                  window=s["window"], sinks=s["sinks"], return_lse=s["lse"], out=s["out"], n_max=s["N"])
        return list(got) if s["lse"] else [got]
    if s["op"] == "mass":
        kernels.attention_mass(s["q"], s["k"], s["lse"], s["scale"], s["mass"], q_len=s["q_len"], kv_len=s["kv_len"],
                               page_table=s["table"], window=s["window"], sinks=s["sinks"], n_max=s["N"])
        return [s["mass"]]
    kernels.kv_evict(s["k"], s["v"], s["mass"], s["kv_len"], s["budget"], s["recent"], sinks=s["sinks"], page_table=s["table"],
                     kv_len_out=s["kv_len_out"], mass_out=s["mass_out"], kept=s["kept"], n_max=s["N"])
    return [s["k"], s["v"], s["mass_out"], s["kept"], s["kv_len_out"]]


# ---- the definition, sequence by sequence and head by head, in 64 bits ----
def _dense64(pool, table, page, b, h, n):
    if table is None:
        return pool[b, h, :n].double()
    at = torch.arange(n, device=pool.device)
    return pool[table[b, at // page].long(), h, at % page].double()


def exact(case, seed):
    s = prepare(case, seed)
    kv, ql = _lengths(case)
    if s["op"] == "evict":
        k, v = s["k"].clone(), s["v"].clone()
        heavy, kept_all = s["mass_out"].double(), s["kept"].clone()
        for b, n in enumerate(kv):
            left = min(n, s["budget"])
            for h in range(s["Hkv"]):
                w = s["mass"][b, h, :n].tolist()
                must = [i for i in range(n) if i < s["sinks"] or i >= n - s["recent"]] if n > left else list(range(n))
                rest = sorted((i for i in range(s["sinks"], n - s["recent"])), key=lambda i: (-w[i], i)) if n > left else []
                idx = torch.tensor(sorted(must + rest[:left - len(must)]), dtype=torch.long, device=k.device)
                to = torch.arange(left, device=k.device)
                for x, y in ((k, s["k"]), (v, s["v"])):
                    if s["table"] is None:
                        x[b, h, :left] = y[b, h, idx]
                    else:
                        row = s["table"][b].long()
                        x[row[to // s["page"]], h, to % s["page"]] = y[row[idx // s["page"]], h, idx % s["page"]]
                heavy[b, h, :n] = 0
                heavy[b, h, :left] = s["mass"][b, h, idx].double()
                kept_all[b, h, :left] = idx.to(torch.int32)
        return [k.double(), v.double(), heavy, kept_all, torch.tensor([min(n, s["budget"]) for n in kv], dtype=torch.int32)]
    q = s["q"] if s["q"].dim() == 4 else s["q"][:, :, None]
    B, Hq, T, D = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    mass = s["mass"].double() if isinstance(s.get("mass"), torch.Tensor) else None
    per = Hq // s["Hkv"]
    for b in range(B):
        n, t = kv[b], ql[b]
        place = torch.arange(n - t, n, device=q.device)[:, None]
        key = torch.arange(n, device=q.device)[None]
        hidden = key > place
        if s["window"]:
            hidden |= (key <= place - s["window"]) & (key >= s["sinks"])
        for hk in range(s["Hkv"]):
            k64 = _dense64(s["k"], s["table"], s["page"], b, hk, n)
            v64 = _dense64(s["v"], s["table"], s["page"], b, hk, n) if s["op"] != "mass" else None
            for h in range(hk * per, (hk + 1) * per):
                a = torch.einsum("td,nd->tn", q[b, h, :t].double(), k64).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
                if s["op"] == "mass":
                    mass[b, hk, :n] += torch.exp(a - s["lse"][b, h, :t].double()[:, None]).sum(0)
                    continue
                z = torch.logsumexp(a, -1)
                w = torch.exp(a - z[:, None])
                lse[b, h, :t] = z
                out[b, h, :t] = torch.einsum("tn,nd->td", w, v64)
                if mass is not None:
                    mass[b, hk, :n] += w.sum(0)
    if s["op"] == "mass":
        return [mass]
    if s["op"] == "decode":
        out, lse = out[:, :, 0], lse[:, :, 0]
    return [out] + ([lse] if s["lse"] else []) + ([mass] if mass is not None else [])
