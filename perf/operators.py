"""Operators of a serving step around the paged KV cache: per-head norm and
rotation of queries and keys (alone, or writing keys and values into their
pages), attention with a sliding window and visible first tokens (a prompt
over dense keys; a few new tokens over a paged cache, on request with the
attention weight that every key received), and eviction from a cache by that
weight.

A case is a dict of sizes and options; `listed()` names the fixed ones and
`draw(rng)` gives more of the same ranges. Inputs are made on the GPU from the
seed alone. `run` computes the plain form of an operator in elementary torch
operations, or with `own` set makes the framework's call. All sizes are this
repository's workloads, tests and benchmark, or generic transformer sizes.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def _ops():
    # The package lives in a directory of the working tree's root (its name
    # has a dash, so it is put on the path rather than imported by name).
    pkg = os.path.join(os.getcwd(), "mtp-engine_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mtp_hip import ops
    return ops


def listed():
    return [
        # One decode step of 8 sequences: the new token's queries and keys are
        # normed and rotated, its key and value go into the paged cache. The
        # smallest call: latency and host work.
        {"name": "rope_decode_write", "kind": "rope", "x": "bf16", "B": 8, "T": 1, "H": 32,
         "Hk": 8, "D": 128, "rot": 128, "interleaved": False, "norm": True, "write": True,
         "L": 2048, "page": 16, "start": 1900},
        # A 4096-token prompt, queries and keys as slices of one projection.
        {"name": "rope_prompt", "kind": "rope", "x": "bf16", "B": 1, "T": 4096, "H": 32, "Hk": 8,
         "D": 128, "rot": 128, "interleaved": False, "norm": True, "write": False, "start": 0},
        # The engine's default dtype, half of each head rotated in pairs, a
        # ragged chunk far into a long context.
        {"name": "rope_chunk_f32", "kind": "rope", "x": "f32", "B": 2, "T": 517, "H": 16,
         "Hk": 16, "D": 64, "rot": 32, "interleaved": True, "norm": True, "write": True,
         "L": 2048, "page": 16, "start": 1200, "far": 100000},
        # A prompt under a sliding window with four first tokens left visible.
        {"name": "prompt_window_bf16", "kind": "prompt", "x": "bf16", "B": 1, "T": 4096,
         "L": 4096, "H": 32, "Hk": 8, "D": 128, "window": 1024, "sinks": 4, "ragged": False},
        # A padded batch of ragged chunks behind earlier context, all of it visible.
        {"name": "prompt_chunk_f16", "kind": "prompt", "x": "f16", "B": 4, "T": 1025, "L": 2049,
         "H": 16, "Hk": 16, "D": 64, "window": None, "sinks": 0, "ragged": True},
        # A long prompt, window of half its length: the largest call.
        {"name": "prompt_long_bf16", "kind": "prompt", "x": "bf16", "B": 1, "T": 8192, "L": 8192,
         "H": 32, "Hk": 8, "D": 128, "window": 4096, "sinks": 16, "ragged": False},
        # The engine's default dtype: a batch of short prompts.
        {"name": "prompt_f32", "kind": "prompt", "x": "f32", "B": 2, "T": 1000, "L": 1000,
         "H": 16, "Hk": 16, "D": 64, "window": 256, "sinks": 1, "ragged": False},
        # Decode of 8 ragged sequences, four query heads to a key head.
        {"name": "decode_bf16", "kind": "decode", "x": "bf16", "B": 8, "T": 1, "L": 4096, "H": 32,
         "Hk": 8, "D": 128, "page": 16, "window": None, "sinks": 0, "weights": False},
        # One sequence with a long cache: few rows, the work lies along the keys.
        {"name": "decode_long_bf16", "kind": "decode", "x": "bf16", "B": 1, "T": 1, "L": 131072,
         "H": 32, "Hk": 8, "D": 128, "page": 16, "window": None, "sinks": 0, "weights": False},
        # The chain verify's five positions per sequence under a window, with
        # the weight that each key received.
        {"name": "chain_window_f16", "kind": "decode", "x": "f16", "B": 8, "T": 5, "L": 16384,
         "H": 32, "Hk": 8, "D": 128, "page": 16, "window": 4096, "sinks": 4, "weights": True},
        # A short cache cut down: latency.
        {"name": "evict_small", "kind": "evict", "x": "bf16", "B": 1, "Hk": 8, "D": 128, "L": 700,
         "page": 16, "keep": 256, "sinks": 4, "recent": 64},
        # Prompts of a batch cut to a quarter before decoding.
        {"name": "evict_prompt", "kind": "evict", "x": "bf16", "B": 4, "Hk": 8, "D": 128,
         "L": 8192, "page": 16, "keep": 2048, "sinks": 4, "recent": 512},
    ]


def _logint(rng, lo, hi, step=1):
    """An integer multiple of step, uniform over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


def _heads(rng, most):
    hk = rng.choice([1, 2, 4, 8, 16])
    g = rng.choice([1, 2, 4, 7, 8])
    return (hk * g, hk) if hk * g <= most else (hk, hk)


def _window(rng, L):
    if rng.random() < 0.4:
        return None, 0
    return _logint(rng, 16, max(17, L)), rng.choice([0, 1, 4, 16])


def draw(rng):
    kind = rng.choice(["rope", "prompt", "prompt", "decode", "decode", "evict"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    H, Hk = _heads(rng, 32)
    D = rng.choice([64, 128])
    if kind == "rope":
        B = _logint(rng, 1, 16)
        T = _logint(rng, 1, 4096 // B)
        c = {"kind": "rope", "x": x, "B": B, "T": T, "H": H, "Hk": Hk, "D": D,
             "rot": rng.choice([D, D, D // 2, D // 4]), "interleaved": rng.random() < 0.3,
             "norm": rng.random() < 0.8, "write": rng.random() < 0.5}
        if c["write"]:
            c["L"] = _logint(rng, T, 4096)
            c["page"] = rng.choice([16, 32, 64])
        c["start"] = rng.randint(0, c["L"] - T) if c["write"] else _logint(rng, 1, 200000)
        return c
    if kind == "prompt":
        B = rng.randint(1, 4)
        most = 2048 if x == "f32" else 4096
        T = _logint(rng, 16, most // B)
        L = T if rng.random() < 0.5 else _logint(rng, T, most)
        w, sinks = _window(rng, L)
        return {"kind": "prompt", "x": x, "B": B, "T": T, "L": L, "H": H, "Hk": Hk, "D": D,
                "window": w, "sinks": sinks, "ragged": rng.random() < 0.4}
    if kind == "decode":
        B = _logint(rng, 1, 16)
        T = 1 if rng.random() < 0.5 else rng.randint(2, 8)
        L = _logint(rng, 64, 65536 // B)
        w, sinks = _window(rng, L)
        return {"kind": "decode", "x": x, "B": B, "T": T, "L": L, "H": H, "Hk": Hk, "D": D,
                "page": rng.choice([16, 32, 64]), "window": w, "sinks": sinks,
                "weights": rng.random() < 0.4}
    B = _logint(rng, 1, 8)
    L = _logint(rng, 128, 32768 // B)
    keep = max(32, int(L * rng.uniform(0.1, 0.6)))
    return {"kind": "evict", "x": x, "B": B, "Hk": Hk, "D": D, "L": L,
            "page": rng.choice([16, 32, 64]), "keep": keep, "sinks": rng.choice([0, 1, 4, 16]),
            "recent": rng.choice([0, keep // 8, keep // 2])}


# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _starts(c):
    """Tokens before the queries of each sequence: the last one fills the
    table, the others are spread down to half of it."""
    B, full = c["B"], c["L"] - c.get("T", 0)
    return [full - (full // 2) * (B - 1 - b) // max(1, B - 1) for b in range(B)]


def _lengths(c):
    """Keys of each sequence of a padded batch, from half of the keys up."""
    B, L = c["B"], c["L"]
    return [L - (L // 2) * (B - 1 - b) // max(1, B - 1) for b in range(B)]


def _table(g, c, n, spare=0):
    """A pool of physical pages a little larger than B tables of n positions
    (and spare further ones) need, and the shuffled tables."""
    B, ps = c["B"], c["page"]
    own_pages = -(-n // ps)
    more = -(-spare // ps)
    P = own_pages + more + max(1, own_pages // 8)
    perm = torch.stack([torch.randperm(P, generator=g, device=DEV) for _ in range(B)])
    table = perm[:, :own_pages].repeat_interleave(ps, dim=1)[:, :n].to(torch.int32).contiguous()
    out = perm[:, own_pages:own_pages + more].repeat_interleave(ps, dim=1)[:, :spare]
    return P, table, out.to(torch.int32).contiguous()


def _pool(g, c, P, dtype):
    shape = (P, c["B"], c["Hk"], c["page"], c["D"])
    return _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = _DT[c["x"]]
    k, B, Hk, D = c["kind"], c["B"], c["Hk"], c["D"]
    s = {"case": c}
    if k == "rope":
        T, H = c["T"], c["H"]
        # the projection's output [B, T, (H + 2 Hk) D], sliced into heads
        qkv = _randn(g, B, T, H + 2 * Hk, D, dtype=dt).transpose(1, 2)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        s["wq"] = 1.0 + 0.1 * _randn(g, D) if c["norm"] else None
        s["wk"] = 1.0 + 0.1 * _randn(g, D) if c["norm"] else None
        i = torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64)
        s["inv_freq"] = (10000.0 ** (-2.0 * i / c["rot"])).float()
        s["start"] = torch.tensor([c["start"]] * B, dtype=torch.int64, device=DEV)
        s["positions"] = None
        if c.get("far"):  # where the tokens stand, when it is not where they are stored
            s["positions"] = c["far"] + torch.arange(T, device=DEV).expand(B, T).contiguous()
        if c["write"]:
            P, s["table"], _ = _table(g, c, c["L"])
            s["kp"], s["vp"] = _pool(g, c, P, dt)
    elif k == "prompt":
        T, L, H = c["T"], c["L"], c["H"]
        s["q"] = _randn(g, B, T, H, D, dtype=dt).transpose(1, 2)
        s["k"] = _randn(g, B, L, Hk, D, dtype=dt).transpose(1, 2)
        s["v"] = _randn(g, B, L, Hk, D, dtype=dt).transpose(1, 2)
        s["lengths"] = torch.tensor(_lengths(c), device=DEV) if c["ragged"] else None
    elif k == "decode":
        T, H = c["T"], c["H"]
        s["q"] = _randn(g, B, T, H, D, dtype=dt).transpose(1, 2)
        P, s["table"], _ = _table(g, c, c["L"])
        s["kp"], s["vp"] = _pool(g, c, P, dt)
        s["start"] = torch.tensor(_starts(c), dtype=torch.int64, device=DEV)
        s["weights"] = None
        if c["weights"]:  # what earlier steps gave
            s["weights"] = torch.rand(B, Hk, c["L"], generator=g, device=DEV)
    elif k == "evict":
        P, s["table"], s["out_table"] = _table(g, c, c["L"], c["keep"])
        s["kp"], s["vp"] = _pool(g, c, P, dt)
        # heavy-tailed, and some keys that received nothing
        w = torch.exp(2.0 * _randn(g, B, Hk, c["L"]))
        s["weights"] = w * (torch.rand(B, Hk, c["L"], generator=g, device=DEV) > 0.05)
        s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int64, device=DEV)
    else:
        raise ValueError(k)
    return s


# ---------------------------------------------------------------------------
# Plain forms
def _rows_of(pages, table, page):
    """[B, Hk, L, D] rows of the pages that the table names."""
    b = torch.arange(table.shape[0], device=DEV)[:, None]
    slot = torch.arange(table.shape[1], device=DEV) % page
    return pages[table.long(), b, :, slot[None, :]].transpose(1, 2)


def _norm_rotate(x, w, c, cos, sin):
    y = x.float()
    if c["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    r, rest = y[..., :c["rot"]], y[..., c["rot"]:]
    if c["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r.chunk(2, -1)
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, rest], -1).to(x.dtype)


def _softmax_pv(q, k, v, see, D):
    """q [B, H, T, D], k / v [B, Hk, L, D], see [B, T, L] -> out and the weight
    of each key over the rows of its head's group [B, Hk, L]."""
    B, H, T, _ = q.shape
    Hk, L = k.shape[1], k.shape[2]
    qf = q.float().reshape(B, Hk, (H // Hk) * T, D)
    sc = qf @ k.float().transpose(-1, -2).contiguous() * (1.0 / math.sqrt(D))
    sc = sc.view(B, Hk, H // Hk, T, L).masked_fill(~see[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(sc - m)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = p.view(B, Hk, -1, L) @ v.float()
    return out.view(B, H, T, D).to(q.dtype), p.sum((2, 3))


def _see(pos, L, c):
    """Which of the keys 0 .. L - 1 a query at position pos [B, T] sees."""
    j = torch.arange(L, device=DEV)
    ok = j <= pos[..., None]
    if c["window"] is not None:
        ok = ok & ((j > pos[..., None] - c["window"]) | (j < c["sinks"]))
    return ok


def _plain(s):
    c = s["case"]
    k, D = c["kind"], c["D"]
    if k == "rope":
        B, T = c["B"], c["T"]
        at = s["start"][:, None] + torch.arange(T, device=DEV)
        pos = at if s["positions"] is None else s["positions"]
        ang = pos.double()[..., None] * s["inv_freq"].double()  # [B, T, rot / 2]
        cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
        q = _norm_rotate(s["q"], s["wq"], c, cos, sin)
        kk = _norm_rotate(s["k"], s["wk"], c, cos, sin)
        if not c["write"]:
            return {"q": q, "k": kk}
        b = torch.arange(B, device=DEV)[:, None]
        page = torch.gather(s["table"].long(), 1, at)
        s["kp"][page, b, :, at % c["page"]] = kk.transpose(1, 2)
        s["vp"][page, b, :, at % c["page"]] = s["v"].transpose(1, 2)
        return {"q": q, "k_pages": s["kp"], "v_pages": s["vp"]}
    if k == "prompt":
        T, L = c["T"], c["L"]
        pos = torch.arange(L - T, L, device=DEV).expand(c["B"], T)
        see = _see(pos, L, c)
        if s["lengths"] is not None:  # padded keys and queries
            n = s["lengths"][:, None, None]
            see = see & (torch.arange(L, device=DEV) < n) & (pos[..., None] < n)
        return _softmax_pv(s["q"], s["k"], s["v"], see, D)[0]
    if k == "decode":
        kk = _rows_of(s["kp"], s["table"], c["page"])
        vv = _rows_of(s["vp"], s["table"], c["page"])
        pos = s["start"][:, None] + torch.arange(c["T"], device=DEV)
        out, w = _softmax_pv(s["q"], kk, vv, _see(pos, c["L"], c), D)
        if s["weights"] is None:
            return out
        s["weights"] += w
        return {"out": out, "weights": s["weights"]}
    B, L, keep = c["B"], c["L"], c["keep"]
    j = torch.arange(L, device=DEV)
    n = s["lengths"][:, None]
    fixed = (j < c["sinks"]) | (j >= n - c["recent"])
    key = s["weights"].double().masked_fill(fixed[:, None], math.inf)
    key = key.masked_fill((j >= n)[:, None], -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    new = s["lengths"].clamp_max(keep)
    live = torch.arange(keep, device=DEV) < new[:, None]  # [B, keep]
    kept = order.masked_fill(~live[:, None], L).sort(-1).values
    at = kept.clamp_max(L - 1)
    w = torch.gather(s["weights"], 2, at).masked_fill(~live[:, None], 0.0)
    b = torch.arange(B, device=DEV)[:, None, None]
    h = torch.arange(c["Hk"], device=DEV)[None, :, None]
    src = s["table"].long()[b, at]
    to = torch.arange(keep, device=DEV) % c["page"]
    dst = s["out_table"].long()[:, None, :]
    sel = live[:, None, :, None]
    s["kp"][dst, b, h, to] = torch.where(sel, s["kp"][src, b, h, at % c["page"]],
                                         s["kp"][dst, b, h, to])
    s["vp"][dst, b, h, to] = torch.where(sel, s["vp"][src, b, h, at % c["page"]],
                                         s["vp"][dst, b, h, to])
    return {"kept": kept.masked_fill(~live[:, None], -1).to(torch.int32), "weights": w,
            "lengths": new, "k_pages": s["kp"], "v_pages": s["vp"]}


def run(s):
    if not own:
        return _plain(s)
    ops = _ops()
    c = s["case"]
    k = c["kind"]
    if k == "rope":
        o = dict(positions=s["positions"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                 norm=c["norm"], interleaved=c["interleaved"])
        if not c["write"]:
            q, kk = ops.qk_norm_rope(s["q"], s["k"], s["inv_freq"], s["start"], **o)
            return {"q": q, "k": kk}
        q = ops.qk_norm_rope_write(s["q"], s["k"], s["v"], s["inv_freq"], s["kp"], s["vp"],
                                   s["table"], s["start"], **o)
        return {"q": q, "k_pages": s["kp"], "v_pages": s["vp"]}
    if k == "prompt":
        return ops.window_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"], s["lengths"])
    if k == "decode":
        out = ops.paged_window_attention(s["q"], s["kp"], s["vp"], s["table"], c["page"],
                                         s["start"], c["window"], c["sinks"],
                                         weights=s["weights"])
        return out if s["weights"] is None else {"out": out, "weights": s["weights"]}
    kept, w, n = ops.kv_evict(s["weights"], s["lengths"], s["kp"], s["vp"], s["table"],
                              s["out_table"], c["sinks"], c["recent"])
    return {"kept": kept, "weights": w, "lengths": n, "k_pages": s["kp"], "v_pages": s["vp"]}


# ---------------------------------------------------------------------------
def _seen(first, T, L, window, sinks, length):
    """Pairs of query and key, and keys that any query sees, of T queries from
    position first on."""
    pairs, hi = 0, min(first + T, L, length)
    for p in range(first, min(first + T, length)):
        lo = 0 if window is None else max(0, p - window + 1)
        pairs += min(p + 1, hi) - lo + (0 if window is None else min(sinks, lo))
    lo = 0 if window is None else max(0, first - window + 1)
    return pairs, max(0, hi - lo) + (0 if window is None else min(sinks, lo))


def work(case):
    c = case
    k, xb, B, Hk, D = c["kind"], _BYTES[c["x"]], c["B"], c["Hk"], c["D"]
    if k == "rope":
        rows = B * c["T"] * (c["H"] + Hk + (Hk if c["write"] else 0))
        return {"bytes": 2 * rows * D * xb + 4 * c["rot"] // 2 + (8 * D if c["norm"] else 0) +
                8 * B + (4 * B * c["T"] if c["write"] else 0), "flops": 8.0 * rows * D}
    if k == "evict":
        rows = sum(min(n, c["keep"]) for n in _lengths(c)) * Hk
        return {"bytes": 4 * sum(_lengths(c)) * Hk + 4 * rows * D * xb + 8 * rows +
                4 * B * 2 * c["keep"], "flops": 0}
    T, L, H = c["T"], c["L"], c["H"]
    if k == "prompt":
        ends = _lengths(c) if c["ragged"] else [L] * B
        seen = [_seen(L - T, T, L, c["window"], c["sinks"], n) for n in ends]
    else:
        seen = [_seen(n, T, L, c["window"], c["sinks"], L) for n in _starts(c)]
    keys = sum(n for _, n in seen)
    extra = 4 * keys if k == "decode" else 0
    if k == "decode" and c["weights"]:
        extra += 8 * keys * Hk
    return {"bytes": 2 * keys * Hk * D * xb + 2 * B * H * T * D * xb + extra,
            "flops": 4.0 * sum(n for n, _ in seen) * H * D}


# ---------------------------------------------------------------------------
# The same from the definitions, in 64 bits
def _exact_rotate(x, w, c, pos, inv_freq):
    x = x.double()
    if c["norm"]:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["D"] + EPS) * w.double()
    half = c["rot"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       pos[:, None, :, None].double() * inv_freq.double())
    i = torch.arange(half, device=DEV)
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attention(q, k, v, first, c, ends):
    """Per sequence and head: only the keys that the queries see at all."""
    B, H, T, D = q.shape
    G = H // k.shape[1]
    out = torch.zeros(B, H, T, D, dtype=torch.float64, device=DEV)
    got = torch.zeros(B, k.shape[1], k.shape[2], dtype=torch.float64, device=DEV)
    for b in range(B):
        n = int(ends[b])
        rows = max(0, min(T, n - int(first[b])))
        if rows <= 0:
            continue
        p = int(first[b]) + torch.arange(rows, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        hidden = j > p
        if c["window"] is not None:
            hidden |= (p - j >= c["window"]) & (j >= c["sinks"])
        for h in range(H):
            kk, vv = k[b, h // G, :n].double(), v[b, h // G, :n].double()
            z = torch.mm(q[b, h, :rows].double(), kk.t().contiguous()) / math.sqrt(D)
            a = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            out[b, h, :rows] = torch.mm(a, vv)
            got[b, h // G, :n] += a.sum(0)
    return out, got


def exact(case, seed):
    s, c = prepare(case, seed), case
    k = c["kind"]
    if k == "rope":
        B, T = c["B"], c["T"]
        at = s["start"][:, None] + torch.arange(T, device=DEV)[None]
        pos = at if s["positions"] is None else s["positions"]
        q = _exact_rotate(s["q"], s["wq"], c, pos, s["inv_freq"])
        kk = _exact_rotate(s["k"], s["wk"], c, pos, s["inv_freq"])
        if not c["write"]:
            return {"q": q, "k": kk}
        kp, vp = s["kp"].double(), s["vp"].double()
        for b in range(B):
            page, slot = s["table"][b, at[b]].long(), at[b] % c["page"]
            kp[page, b, :, slot] = kk[b].transpose(0, 1)
            vp[page, b, :, slot] = s["v"][b].transpose(0, 1).double()
        return {"q": q, "k_pages": kp, "v_pages": vp}
    if k == "prompt":
        first = [c["L"] - c["T"]] * c["B"]
        ends = _lengths(c) if c["ragged"] else [c["L"]] * c["B"]
        return _exact_attention(s["q"], s["k"], s["v"], first, c, ends)[0]
    if k == "decode":
        L = c["L"]
        rows = [[p[s["table"][b].long(), b, :, torch.arange(L, device=DEV) % c["page"]]
                 for b in range(c["B"])] for p in (s["kp"], s["vp"])]
        kk, vv = (torch.stack(r).transpose(1, 2) for r in rows)
        out, got = _exact_attention(s["q"], kk, vv, _starts(c), c, [L] * c["B"])
        if s["weights"] is None:
            return out
        return {"out": out, "weights": s["weights"].double() + got}
    kp, vp = s["kp"].double(), s["vp"].double()
    w = torch.zeros(c["B"], c["Hk"], c["keep"], dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lengths(c)):
        m = min(n, c["keep"])
        to, slot = s["out_table"][b, :m].long(), torch.arange(m, device=DEV) % c["page"]
        for h in range(c["Hk"]):
            x = s["weights"][b, h, :n].double().clone()
            x[:c["sinks"]] = math.inf
            x[max(0, n - c["recent"]):] = math.inf
            # the m-th largest; of those that equal it, the first ones fill up
            last = torch.sort(x, descending=True).values[m - 1]
            over, same = x > last, x == last
            fill = same & (torch.cumsum(same, 0) <= m - over.sum())
            idx = torch.nonzero(over | fill)[:, 0]
            w[b, h, :m] = s["weights"][b, h, idx].double()
            page = s["table"][b, idx].long()
            kp[to, b, h, slot] = s["kp"][page, b, h, idx % c["page"]].double()
            vp[to, b, h, slot] = s["vp"][page, b, h, idx % c["page"]].double()
    return {"kept": None, "weights": w, "lengths": None, "k_pages": kp, "v_pages": vp}
