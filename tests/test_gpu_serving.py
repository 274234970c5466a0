"""GPU tests of the serving operators around the paged cache against their
definitions in 64 bits (oracle/serving.py): per-head norm with rotation (alone
and into the pages), windowed attention of prompts and over the paged cache
with the weight of each key, eviction, and a step of all of them.

Error bounds, elementwise, with u = 2^-24 and h = half a step of the output's
type (finfo.eps / 2):
 * norm and rotation: a component is a cos t -+ b sin t of normed a, b. The
   sum of squares, rsqrt, the norm's two products, the reduced angle (its
   rounding is at most pi u), sin / cos (2 ulp) and the last product and sum
   are together below 24 u (|a| + |b|); plus h |y| for the output.
 * attention: a score is off by at most e = (D + 4) u sum |q k| scale + 2 u of
   the exponent's size, which that sum bounds as well: a factor 1 + 2 e on a
   probability, 4 u for its exp2, n u for sums over n keys. 16-bit kernels
   round p to their type once (h). So |out - ref| <= h |ref| + (h16 + 2 e +
   (n + 8) u) sum p |v|, with n the keys of the row and h16 = 0 for fp32.
 * weights: the same factor on each p, plus u of the total for the addition.
"""
import math

import pytest
import torch

from oracle import serving as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half(dt):
    return torch.finfo(dt).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


def within(y, ref, bound, what=""):
    y = y.detach().cpu().double()
    assert y.shape == ref.shape, (y.shape, ref.shape)
    assert torch.isfinite(y).all(), f"{what}: not finite"
    over = ((y - ref).abs() / (bound + 1e-300)).max().item() if y.numel() else 0.0
    assert over <= 1.0, f"{what}: {over:.3g} times the bound"


def inv_freq(rot, base=10000.0, dtype=F32):
    i = torch.arange(rot // 2, dtype=torch.float64)
    return (base ** (-2.0 * i / max(rot, 1))).to(dtype)


# ---------------------------------------------------------------------------
# norm and rotation
def rope_bound(ref, mag, dt):
    return half(dt) * ref.abs() + 24 * U * mag + (1e-7 if dt is F16 else 1e-38)


ROPE = [
    # dtype, B, T, H, Hk, D, rot, interleaved, norm
    (BF16, 8, 1, 32, 8, 128, 128, False, True),
    (BF16, 1, 1, 1, 1, 64, 64, False, True),
    (F16, 2, 37, 7, 1, 64, 32, False, True),
    (F32, 2, 5, 16, 16, 64, 32, True, True),
    (F32, 3, 9, 4, 2, 128, 128, False, False),
    (BF16, 1, 300, 8, 8, 128, 64, True, True),
    (F16, 1, 3, 4, 4, 256, 256, False, True),
    (BF16, 2, 4, 3, 1, 96, 96, False, True),
    (BF16, 2, 4, 3, 1, 80, 16, False, True),
    (BF16, 1, 6, 2, 2, 50, 50, False, True),     # no whole 16 bytes
    (F32, 1, 6, 2, 2, 33, 10, True, True),
    (F16, 1, 2, 2, 1, 128, 0, False, True),      # norm alone
    (F32, 1, 2, 2, 1, 1, 0, False, True),
    (BF16, 1, 2, 1, 1, 512, 8, False, True),     # halves inside one 16-byte chunk
    (F32, 1, 2, 1, 1, 512, 512, False, True),    # more lanes than a wave
    (BF16, 0, 4, 2, 2, 64, 64, False, True),
    (BF16, 2, 0, 2, 2, 64, 64, False, True),
]


@pytest.mark.parametrize("dt,B,T,H,Hk,D,rot,inter,norm", ROPE)
@pytest.mark.parametrize("layout", ["slices", "dense"])
def test_qk_norm_rope(dt, B, T, H, Hk, D, rot, inter, norm, layout):
    from mtp_hip import ops
    g = gen(D + T)
    if layout == "slices":  # one projection's output, sliced into heads
        x = randn(g, B, T, H + 2 * Hk, D, dtype=dt).transpose(1, 2)
        q, k = x[:, :H], x[:, H:H + Hk]
        xd = x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
        qd, kd = xd[:, :H], xd[:, H:H + Hk]
    else:
        q, k = randn(g, B, H, T, D, dtype=dt), randn(g, B, Hk, T, D, dtype=dt)
        qd, kd = q.to(DEV), k.to(DEV)
    wq, wk = 1 + 0.1 * randn(g, D), 1 + 0.1 * randn(g, D)
    f = inv_freq(rot)
    pos = torch.randint(0, 200000, (B, T), generator=g)
    print(f"case rope {dt} {(B, T, H, Hk, D, rot, inter, norm, layout)}", flush=True)
    qo, ko = ops.qk_norm_rope(qd, kd, f.to(DEV), positions=pos.to(DEV), q_weight=wq.to(DEV),
                              k_weight=wk.to(DEV), norm=norm, interleaved=inter)
    assert qo.dtype == dt and ko.dtype == dt
    for y, x, w in ((qo, q, wq), (ko, k, wk)):
        ref, mag = S.norm_rotate(x, w, pos, f, norm=norm, interleaved=inter)
        within(y, ref, rope_bound(ref, mag, dt))
    if layout == "slices" and B and T > 1 and H > 1:
        assert qo.transpose(1, 2).is_contiguous()  # the inputs' order of dimensions


@pytest.mark.parametrize("start", ["host", "shared", "per_row"])
def test_qk_norm_rope_positions_follow_start(start):
    from mtp_hip import ops
    g = gen(3)
    B, T, H, Hk, D = 3, 4, 4, 2, 64
    q, k = randn(g, B, H, T, D), randn(g, B, Hk, T, D)
    f = inv_freq(D, dtype=torch.float64)
    at = {"host": [11] * 3, "shared": [2 ** 20] * 3, "per_row": [0, 5, 131071]}[start]
    arg = 11 if start == "host" else torch.tensor(at if start == "per_row" else at[:1]).to(DEV)
    qo, ko = ops.qk_norm_rope(q.to(DEV), k.to(DEV), f.to(DEV), arg)
    pos = torch.tensor(at)[:, None] + torch.arange(T)
    for y, x in ((qo, q), (ko, k)):
        ref, mag = S.norm_rotate(x, None, pos, f)
        within(y, ref, rope_bound(ref, mag, F32))


def test_qk_norm_rope_extremes():
    """Zero rows, huge and tiny values, one position shared by the batch."""
    from mtp_hip import ops
    D = 128
    x = torch.zeros(1, 4, 2, D)
    x[0, 1] = 1e18
    x[0, 2] = 1e-18
    x[0, 3, :, 0] = 3.0
    pos = torch.tensor([7, 9])
    f = inv_freq(D)
    qo, ko = ops.qk_norm_rope(x.to(DEV), x.to(DEV), f.to(DEV), positions=pos.to(DEV))
    ref, mag = S.norm_rotate(x, None, pos[None], f)
    within(qo, ref, rope_bound(ref, mag, F32) + 1e-30)
    assert torch.equal(qo, ko)
    # a NaN stays in its row
    x[0, 0, 0, 5] = math.nan
    qo, _ = ops.qk_norm_rope(x.to(DEV), x.to(DEV), f.to(DEV), positions=pos.to(DEV))
    assert torch.isnan(qo[0, 0, 0]).all() and torch.isfinite(qo[0, 0, 1]).all()
    assert torch.isfinite(qo[0, 1:]).all()


def make_pages(g, P, B, Hk, ps, D, L, dtype, spare=0):
    kp, vp = randn(g, P, B, Hk, ps, D, dtype=dtype), randn(g, P, B, Hk, ps, D, dtype=dtype)
    n = -(-L // ps)
    m = -(-spare // ps)
    assert n + m <= P
    perm = torch.stack([torch.randperm(P, generator=g) for _ in range(B)])
    table = perm[:, :n].repeat_interleave(ps, dim=1)[:, :L].to(torch.int32)
    out = perm[:, n:n + m].repeat_interleave(ps, dim=1)[:, :spare].to(torch.int32)
    return kp, vp, table.contiguous(), out.contiguous()


@pytest.mark.parametrize("dt,D,ps", [(BF16, 128, 16), (F16, 64, 32), (F32, 64, 16), (F32, 20, 5),
                                     (BF16, 50, 7)])
def test_qk_norm_rope_write(dt, D, ps):
    from mtp_hip import ops
    g = gen(D)
    B, T, H, Hk, L, P = 3, 5, 6, 2, 60, 16
    x = randn(g, B, T, H + 2 * Hk, D, dtype=dt).transpose(1, 2)
    q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    kp, vp, table, _ = make_pages(g, P, B, Hk, ps, D, L, dt)
    table[1, 30:] = -1        # unmapped
    table[2, 9] = P           # outside the pool
    start = torch.tensor([0, 28, 7])
    wq, wk = 1 + 0.1 * randn(g, D), 1 + 0.1 * randn(g, D)
    f = inv_freq(D)
    depth = torch.tensor([0, 1, 1, 2, 2])  # tree nodes: angles apart from slots
    xd = x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    kd, vd = kp.to(DEV), vp.to(DEV)
    for positions in (None, depth):
        qo = ops.qk_norm_rope_write(
            xd[:, :H], xd[:, H:H + Hk], xd[:, H + Hk:], f.to(DEV), kd, vd, table.to(DEV),
            start.to(DEV), positions=None if positions is None else positions.to(DEV),
            q_weight=wq.to(DEV), k_weight=wk.to(DEV))
        at = start[:, None] + torch.arange(T)
        pos = at if positions is None else positions[None].expand(B, T)
        ref, mag = S.norm_rotate(q, wq, pos, f)
        within(qo, ref, rope_bound(ref, mag, dt))
        ref, mag = S.norm_rotate(k, wk, pos, f)
        touched = torch.zeros(P, B, ps, dtype=torch.bool)
        for b in range(B):
            for t in range(T):
                p = int(at[b, t])
                pid = int(table[b, p]) if p < L else -1
                if 0 <= pid < P:
                    touched[pid, b, p % ps] = True
                    within(kd[pid, b, :, p % ps], ref[b, :, t],
                           rope_bound(ref[b, :, t], mag[b, :, t], dt))
                    assert torch.equal(vd[pid, b, :, p % ps].cpu(), v[b, :, t])
        idle = ~touched[:, :, None, :, None].expand_as(kp)
        assert torch.equal(kd.cpu()[idle], kp[idle]) and torch.equal(vd.cpu()[idle], vp[idle])


# ---------------------------------------------------------------------------
# windowed attention
def attn_check(y, q, k, v, see, dt, what="", rounded=True):
    ref, spread, w, score = S.attention(q, k, v, see)
    n = see.sum(-1)[:, None, :, None].double()
    e = (q.shape[-1] + 6) * U * score[..., None]
    h16 = half(dt) if dt is not F32 and rounded else 0.0
    bound = half(dt) * ref.abs() + (h16 + 2 * e + (n + 12) * U) * spread + \
        (2.0 ** -25 * (spread > 0) if dt is F16 else 0.0)  # subnormal p and outputs
    empty = ~see.any(-1)
    y = y.detach().cpu()
    assert (y.transpose(1, 2)[empty] == 0).all(), f"{what}: a row without keys is not zero"
    within(y, ref, bound, what)
    return w, e


PROMPT = [
    # dtype, B, T, L, H, Hk, D, window, sinks
    (BF16, 1, 1, 1, 1, 1, 64, None, 0),
    (BF16, 1, 1, 40, 4, 1, 128, None, 0),
    (BF16, 2, 33, 33, 4, 2, 64, None, 0),
    (F16, 1, 129, 129, 2, 2, 128, None, 0),
    (BF16, 1, 200, 321, 7, 1, 128, 50, 3),
    (BF16, 2, 64, 300, 8, 8, 64, 64, 4),
    (F16, 1, 257, 257, 8, 2, 64, 1, 0),       # a window of the query itself
    (F16, 1, 100, 100, 2, 1, 128, 1, 1),
    (BF16, 1, 300, 300, 4, 4, 128, 31, 40),   # sinks and window meet
    (BF16, 1, 513, 513, 2, 2, 64, 1000, 4),   # window past the prompt
    (BF16, 1, 130, 700, 4, 2, 128, 128, 0),
    (F32, 1, 1, 77, 4, 2, 64, None, 0),
    (F32, 2, 70, 70, 4, 2, 64, 16, 1),
    (F32, 1, 150, 200, 2, 2, 128, None, 0),
    (F32, 1, 64, 128, 6, 2, 128, 33, 16),
    (BF16, 1, 37, 50, 3, 1, 80, 20, 2),       # other head sizes
    (F16, 1, 20, 20, 2, 2, 33, None, 0),
    (F32, 1, 20, 30, 2, 1, 5, 7, 1),
    (BF16, 1, 9, 70, 2, 1, 256, 30, 2),
    (F32, 1, 5, 9, 1, 1, 1000, None, 0),
    (BF16, 0, 5, 9, 2, 1, 64, None, 0),
    (BF16, 1, 0, 9, 2, 1, 64, None, 0),
    (BF16, 1, 0, 0, 2, 1, 64, None, 0),
]


@pytest.mark.parametrize("dt,B,T,L,H,Hk,D,window,sinks", PROMPT)
@pytest.mark.parametrize("layout", ["bthd", "bhtd"])
def test_window_attention(dt, B, T, L, H, Hk, D, window, sinks, layout):
    from mtp_hip import ops
    g = gen(T * 7 + L)
    q, k, v = (randn(g, B, h, n, D, dtype=dt) for h, n in ((H, T), (Hk, L), (Hk, L)))
    dev = [x.to(DEV) for x in (q, k, v)]
    if layout == "bthd":
        dev = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in dev]
    print(f"case prompt {dt} {(B, T, L, H, Hk, D, window, sinks, layout)}", flush=True)
    out = ops.window_attention(*dev, window, sinks)
    see = S.visible([L - T] * B, [T] * B, T, L, window, sinks)
    attn_check(out, q, k, v, see, dt)


@pytest.mark.parametrize("dt,T,L,D,window,sinks", [
    (BF16, 150, 150, 64, None, 0), (BF16, 70, 200, 128, 40, 4), (F32, 60, 90, 64, 20, 1),
    (F16, 40, 300, 128, None, 0), (BF16, 30, 60, 40, 16, 2)])
def test_window_attention_padded_batch(dt, T, L, D, window, sinks):
    """Ragged lengths, an empty sequence among them, and garbage behind them."""
    from mtp_hip import ops
    g = gen(L)
    n = [L, L - 1, L - T + 1, L - T, 5, 0, 2 * L, -3]
    B, H, Hk = len(n), 4, 2
    q, k, v = (randn(g, B, h, m, D, dtype=dt) for h, m in ((H, T), (Hk, L), (Hk, L)))
    ends = [min(max(x, 0), L) for x in n]
    for b in range(B):
        k[b, :, ends[b]:] = math.nan
        v[b, :, ends[b]:] = math.inf
        q[b, :, max(0, ends[b] - (L - T)):] = math.nan
    out = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window, sinks,
                               lengths=torch.tensor(n).to(DEV))
    see = S.visible([L - T] * B, [max(0, e - (L - T)) for e in ends], T, L, window, sinks)
    qz = torch.nan_to_num(q)
    attn_check(out, qz, k.nan_to_num(), v.nan_to_num(posinf=0.0), see, dt)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (BF16, 128), (F16, 128), (F32, 64), (F32, 40)])
def test_hidden_keys_never_reach_a_row(dt, D):
    """Infinite and NaN keys and values that some rows see and others do not."""
    from mtp_hip import ops
    g = gen(9)
    B, H, Hk, T, window, sinks = 1, 2, 1, 170, 20, 2
    q, k, v = (randn(g, B, h, T, D, dtype=dt) for h in (H, Hk, Hk))
    v[0, 0, 100, 3] = math.nan
    v[0, 0, 140, 5] = math.inf
    k[0, 0, 60, 7] = math.nan
    out = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window, sinks).cpu()
    see = S.visible([0], [T], T, T, window, sinks)
    hit = see[0][:, [60, 100, 140]].any(-1)
    clean = out[:, :, ~hit]
    ref = S.attention(q[:, :, ~hit], k.nan_to_num(), v.nan_to_num(posinf=0.0), see[:, ~hit])
    assert torch.isfinite(clean).all()
    bound = 2 * half(dt) * (ref[0].abs() + ref[1]) + 1e-3 * U + 400 * U * ref[1] * (1 + ref[3])[..., None]
    within(clean, ref[0], bound)
    # rows that see them: NaN where the sum is
    assert torch.isnan(out[0, :, 100:120, 3]).all()
    assert torch.isinf(out[0, :, 140:160, 5]).all()
    assert torch.isnan(out[0, :, 60:80]).all()
    assert torch.isfinite(out[0, :, 105:120, 4]).all()


def test_window_attention_large_scores():
    """Scores of some hundreds and an explicit scale: the maximum carries it."""
    from mtp_hip import ops
    g = gen(4)
    for dt in (BF16, F32):
        q, k, v = (randn(g, 1, 2, 90, 64, dtype=dt) for _ in range(3))
        out = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), scale=12.0)
        see = S.visible([0], [90], 90, 90, None, 0)
        ref, spread, _, score = S.attention(q, k, v, see, scale=12.0)
        e = 70 * U * score[..., None]
        b = half(dt) * ref.abs() + ((half(dt) if dt is not F32 else 0) + 2 * e + 110 * U) * spread
        within(out, ref, b)


DECODE = [
    # dtype, B, T, L, H, Hk, D, page, window, sinks
    (BF16, 1, 1, 1, 1, 1, 64, 16, None, 0),
    (BF16, 8, 1, 300, 8, 2, 128, 16, None, 0),
    (BF16, 2, 5, 333, 8, 2, 128, 16, None, 0),
    (F16, 3, 5, 400, 8, 8, 64, 32, 64, 4),
    (BF16, 1, 1, 5000, 4, 1, 128, 16, None, 0),
    (BF16, 1, 3, 5000, 7, 1, 64, 64, 1000, 16),
    (BF16, 2, 8, 700, 8, 1, 128, 16, 100, 1),   # 64 rows to a key head
    (F16, 1, 17, 600, 14, 2, 64, 16, None, 0),  # 119 rows
    (F32, 2, 1, 600, 4, 4, 64, 16, None, 0),
    (F32, 2, 4, 257, 8, 2, 128, 32, 31, 2),
    (F32, 1, 1, 3000, 2, 1, 128, 16, None, 0),
    (BF16, 2, 3, 90, 3, 1, 80, 7, 20, 2),       # other head and page sizes
    (F32, 1, 2, 40, 2, 1, 6, 5, None, 0),
    (BF16, 2, 40, 100, 2, 2, 64, 16, 16, 4),    # more queries than a window
]


@pytest.mark.parametrize("dt,B,T,L,H,Hk,D,page,window,sinks", DECODE)
@pytest.mark.parametrize("weights", [False, True])
def test_paged_window_attention(dt, B, T, L, H, Hk, D, page, window, sinks, weights):
    from mtp_hip import ops
    g = gen(L + T)
    P = -(-L // page) + 3
    kp, vp, table, _ = make_pages(g, P, B, Hk, page, D, L, dt)
    q = randn(g, B, T, H, D, dtype=dt).transpose(1, 2)
    first = [max(0, L - T - 37 * b) for b in range(B)]
    w = torch.rand(B, Hk, L, generator=g) if weights else None
    wd = w.to(DEV) if weights else None
    print(f"case paged {dt} {(B, T, L, H, Hk, D, page, window, sinks, weights)}", flush=True)
    out = ops.paged_window_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV), page,
                                     torch.tensor(first).to(DEV), window, sinks, weights=wd)
    kk, _ = S.rows_of(kp, table, page)
    vv, _ = S.rows_of(vp, table, page)
    see = S.visible(first, [T] * B, T, L, window, sinks)
    got, e = attn_check(out, q, kk, vv, see, dt)
    if weights:
        total = w.double() + got
        within(wd, total, U * total * 2 + (2 * e.max() + (L + 24 + H // Hk * T) * U) * got + 1e-37)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F32, 64), (BF16, 24)])
def test_paged_window_attention_empty_and_edge_rows(dt, D):
    """Starts before the cache, at its end and past it; unmapped pages; garbage
    in slots that nobody sees."""
    from mtp_hip import ops
    g = gen(5)
    B, T, L, H, Hk, page, P, window, sinks = 7, 3, 100, 4, 2, 16, 9, 24, 2
    kp, vp, table, _ = make_pages(g, P, B, Hk, page, D, L, dt)
    first = [-3, -1, 0, 97, 100, 130, 10 ** 12]
    table[3, 80:90] = -1
    table[3, 0] = P + 5
    kk, ok = S.rows_of(kp, table, page)
    vv, _ = S.rows_of(vp, table, page)
    see = S.visible(first, [T] * B, T, L, window, sinks) & ok[:, None]
    unseen = ~see.any(1)
    for b in range(B):
        for j in range(L):
            if unseen[b, j] and 0 <= int(table[b, j]) < P:
                kp[int(table[b, j]), b, :, j % page] = math.nan
                vp[int(table[b, j]), b, :, j % page] = math.inf
    q = randn(g, B, H, T, D, dtype=dt)
    w = torch.zeros(B, Hk, L, device=DEV)
    out = ops.paged_window_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV), page,
                                     torch.tensor(first).to(DEV), window, sinks, weights=w)
    got, e = attn_check(out, q, kk, vv, see, dt)
    within(w, got, 2 * U * got + (2 * e.max() + (L + 30) * U) * got + 1e-37)
    assert (w.cpu()[unseen[:, None].expand_as(w)] == 0).all()
    # without a window a start past the table sees all of it
    out = ops.paged_window_attention(q[:1].to(DEV), kp[:, 3:4].contiguous().to(DEV),
                                     vp[:, 3:4].contiguous().to(DEV), table[4:5].to(DEV) * 0, page,
                                     10 ** 12)
    assert out.shape == (1, H, T, D)


def test_paged_window_attention_hidden_values():
    """A NaN value under the window's edge of some of the rows of one call."""
    from mtp_hip import ops
    g = gen(6)
    for dt, D in ((BF16, 128), (F16, 64), (F32, 64)):
        B, T, L, H, Hk, page = 1, 5, 2000, 4, 1, 16
        kp, vp, table, _ = make_pages(g, 130, B, Hk, page, D, L, dt)
        first, window = [1990], 500
        bad = 1990 - 500 + 2  # queries 0 and 1 see it, 2 .. 4 do not
        vp[int(table[0, bad]), 0, 0, bad % page, 9] = math.nan
        q = randn(g, B, H, T, D, dtype=dt)
        out = ops.paged_window_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV), page,
                                         torch.tensor(first).to(DEV), window, 4).cpu()
        assert torch.isnan(out[0, :, :2, 9]).all() and torch.isfinite(out[0, :, :2, 10]).all()
        kk, vv = S.rows_of(kp, table, page)[0], S.rows_of(vp, table, page)[0]
        see = S.visible(first, [T], T, L, window, 4)
        attn_check(out[:, :, 2:], q[:, :, 2:], kk, vv, see[:, 2:], dt)


# ---------------------------------------------------------------------------
# eviction
EVICT = [
    # dtype, B, Hk, L, D, page, keep, sinks, recent, lengths
    (BF16, 2, 3, 100, 64, 16, 40, 4, 10, [100, 57]),
    (F32, 1, 1, 1, 8, 4, 1, 0, 0, [1]),
    (BF16, 3, 2, 64, 128, 16, 64, 0, 0, [64, 30, 0]),   # nothing to drop
    (F16, 1, 2, 3000, 64, 32, 777, 0, 0, [2999]),
    (BF16, 2, 1, 2500, 64, 16, 1030, 16, 1000, [2500, 1031]),
    (F32, 1, 2, 90, 5, 7, 30, 10, 20, [90]),            # forced entries alone
    (BF16, 1, 1, 50, 3, 4, 20, 1, 1, [70]),             # a length past the table
    (torch.float8_e4m3fn, 1, 2, 200, 64, 16, 33, 2, 8, [200]),
]


@pytest.mark.parametrize("dt,B,Hk,L,D,page,keep,sinks,recent,lengths", EVICT)
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_kv_evict(dt, B, Hk, L, D, page, keep, sinks, recent, lengths, kind):
    from mtp_hip import ops
    g = gen(L)
    P = -(-L // page) + -(-keep // page) + 2
    kp, vp, table, out_table = make_pages(g, P, B, Hk, page, D, L, F32 if dt.itemsize == 1 else dt,
                                          keep)
    kp, vp = kp.to(dt), vp.to(dt)
    w = torch.exp(2 * torch.randn(B, Hk, L, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, (B, Hk, L), generator=g).float()
    if kind == "odd":
        w = torch.randn(B, Hk, L, generator=g)
        pick = torch.randint(0, 12, w.shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42)):
            w[pick == i] = x
        table[:, L // 3:L // 2] = -1
        table[0, -1] = P
    kd, vd = kp.to(DEV), vp.to(DEV)
    print(f"case evict {dt} {(B, Hk, L, D, page, keep, sinks, recent, kind)}", flush=True)
    kept, ow, n = ops.kv_evict(w.to(DEV), torch.tensor(lengths).to(DEV), kd, vd, table.to(DEV),
                               out_table.to(DEV), sinks, recent)
    rk, rw, rn, rkp, rvp = S.evict(w, lengths, kp, vp, table, out_table, sinks, recent)
    assert torch.equal(kept.cpu(), rk) and torch.equal(n.cpu(), rn)
    assert torch.equal(ow.cpu().view(torch.int32), rw.view(torch.int32))
    raw = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[dt.itemsize]
    assert torch.equal(kd.cpu().view(raw), rkp.view(raw))
    assert torch.equal(vd.cpu().view(raw), rvp.view(raw))


def test_kv_evict_long_cache():
    """Tens of thousands of entries, many of them equal, against a stable sort."""
    from mtp_hip import ops
    g = gen(11)
    B, Hk, L, keep = 1, 2, 40001, 9001
    w = torch.randint(0, 5000, (B, Hk, L), generator=g).float() / 64
    P = L // 64 + keep // 64 + 4
    kp, vp, table, out_table = make_pages(g, P, B, Hk, 64, 2, L, BF16, keep)
    kd, vd = kp.to(DEV), vp.to(DEV)
    kept, ow, n = ops.kv_evict(w.to(DEV), torch.tensor([L]).to(DEV), kd, vd, table.to(DEV),
                               out_table.to(DEV), 4, 100)
    key = w.double()
    key[..., :4] = key[..., -100:] = math.inf
    ref = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    assert torch.equal(kept.cpu().long(), ref) and int(n) == keep
    assert torch.equal(ow.cpu(), torch.gather(w, 2, ref))
    for h in range(Hk):
        src = kp[table[0, ref[0, h]].long(), 0, h, ref[0, h] % 64]
        to = torch.arange(keep)
        assert torch.equal(kd.cpu()[out_table[0].long(), 0, h, to % 64], src)


# ---------------------------------------------------------------------------
# together
def _layer(dt, B, H, Hk, D, L, page, keep, T, g):
    P = -(-L // page) + -(-keep // page) + 1
    kp, vp, table, out_table = make_pages(g, P, B, Hk, page, D, L, dt, keep)
    n = H + 2 * Hk
    prompt = randn(g, B, T, n, D, dtype=dt).transpose(1, 2)
    steps = [randn(g, B, 2, n, D, dtype=dt).transpose(1, 2) for _ in range(3)]
    return kp, vp, table, out_table, prompt, steps


@pytest.mark.parametrize("dt", [BF16, F32])
def test_prompt_then_decode_then_evict(dt):
    """A prompt through its dense attention and into the pages, two-token steps
    over the cache, an eviction, and a step over what is left."""
    from mtp_hip import ops
    g = gen(12)
    B, H, Hk, D, L, page, keep, T, window, sinks = 2, 8, 2, 64, 160, 16, 48, 100, 64, 4
    kp, vp, table, out_table, prompt, steps = _layer(dt, B, H, Hk, D, L, page, keep, T, g)
    wq, wk = 1 + 0.1 * randn(g, D), 1 + 0.1 * randn(g, D)
    f = inv_freq(D)
    kd, vd, td = kp.to(DEV), vp.to(DEV), table.to(DEV)
    opt = dict(q_weight=wq.to(DEV), k_weight=wk.to(DEV))
    kv_len = torch.zeros(B, dtype=torch.int64, device=DEV)
    weights = torch.zeros(B, Hk, L, device=DEV)

    def split(x):
        return x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]

    q, k, v = split(prompt.to(DEV))
    qr, kr = ops.qk_norm_rope(q, k, f.to(DEV), kv_len, **opt)
    out = ops.window_attention(qr, kr, v, window, sinks)
    see = S.visible([0] * B, [T] * B, T, T, window, sinks)
    attn_check(out, qr.cpu(), kr.cpu(), split(prompt)[2], see, dt, "prompt")
    q2 = ops.qk_norm_rope_write(q, k, v, f.to(DEV), kd, vd, td, kv_len, **opt)
    assert torch.equal(q2, qr)
    # the same rows by the paged entry: same keys, same answer within the bounds
    paged = ops.paged_window_attention(qr, kd, vd, td, page, kv_len, window, sinks, weights=weights)
    kk, vv = S.rows_of(kd, table, page)[0], S.rows_of(vd, table, page)[0]
    assert torch.equal(kk[:, :, :T], kr.cpu())
    attn_check(paged, qr.cpu(), kk, vv, S.visible([0] * B, [T] * B, T, L, window, sinks), dt)
    kv_len += T
    total = S.attention(qr.cpu(), kk, vv, S.visible([0] * B, [T] * B, T, L, window, sinks))[2]
    for i, x in enumerate(steps[:2]):
        q, k, v = split(x.to(DEV))
        qr = ops.qk_norm_rope_write(q, k, v, f.to(DEV), kd, vd, td, kv_len, **opt)
        out = ops.paged_window_attention(qr, kd, vd, td, page, kv_len, window, sinks,
                                         weights=weights)
        at = [T + 2 * i] * B
        kk, vv = S.rows_of(kd, table, page)[0], S.rows_of(vd, table, page)[0]
        see = S.visible(at, [2] * B, 2, L, window, sinks)
        attn_check(out, qr.cpu(), kk, vv, see, dt, f"step {i}")
        total += S.attention(qr.cpu(), kk, vv, see)[2]
        kv_len += 2
    # each p is within the attention's factor (scores of normed rows stay
    # below 8 sqrt(D)), summed over at most G * T rows a call and three calls
    within(weights, total, (2 * 70 * U * 8 * 8 + 1000 * U) * total + 1e-30)
    before = (kd.cpu().clone(), vd.cpu().clone())
    kept, w, n = ops.kv_evict(weights, kv_len, kd, vd, td, out_table.to(DEV), sinks, 16)
    rk, rw, rn, rkp, rvp = S.evict(weights.cpu(), kv_len.cpu().tolist(), *before, table, out_table,
                                   sinks, 16)
    assert torch.equal(kept.cpu(), rk) and torch.equal(n.cpu(), rn) and n.tolist() == [keep] * B
    assert torch.equal(kd.cpu(), rkp) and torch.equal(vd.cpu(), rvp)
    q, k, v = split(steps[2].to(DEV))
    out = ops.paged_window_attention(ops.qk_norm_rope(q, k, f.to(DEV), kv_len, **opt)[0], kd, vd,
                                     out_table.to(DEV), page, n)
    qr = ops.qk_norm_rope(q, k, f.to(DEV), kv_len, **opt)[0].cpu()
    kk, vv = S.rows_of(kd, out_table, page)[0], S.rows_of(vd, out_table, page)[0]
    attn_check(out, qr, kk, vv, S.visible([keep] * B, [2] * B, 2, keep, None, 0), dt, "cut")


def test_step_captured_and_replayed():
    """A decode step of all the operators as a graph: the device-held length
    moves on, other inputs come in, eager work runs between the replays."""
    from mtp_hip import _lib, ops
    g = gen(13)
    B, H, Hk, D, L, page, keep, T, window, sinks = 2, 8, 2, 128, 4000, 16, 500, 2, 3000, 4
    dt = BF16
    kp, vp, table, out_table, _, steps = _layer(dt, B, H, Hk, D, L, page, keep, T, g)
    f = inv_freq(D).to(DEV)
    td, od = table.to(DEV), out_table.to(DEV)

    def run(x, kd, vd, kv_len, weights):
        q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
        qr = ops.qk_norm_rope_write(q, k, v, f, kd, vd, td, kv_len)
        out = ops.paged_window_attention(qr, kd, vd, td, page, kv_len, window, sinks,
                                         weights=weights)
        dense = ops.window_attention(qr, qr[:, ::H // Hk], qr[:, ::H // Hk], 1)
        return (out, dense) + ops.kv_evict(weights, kv_len, kd, vd, td, od, sinks, 100)

    def state():
        return (kp.to(DEV), vp.to(DEV), torch.tensor([3900, 2500]).to(DEV),
                torch.zeros(B, Hk, L, device=DEV))

    eager, want = state(), []
    for x in steps:
        want.append([t.cpu() for t in run(x.to(DEV), *eager)])
        eager[2].add_(T)
    st, x = state(), steps[0].to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, *state())
        _lib.reserve_workspace(torch.device(DEV), 1 << 26)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = run(x, *st)
        st[2].add_(T)
    for i, step in enumerate(steps):
        x.copy_(step)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want[i]):
            assert torch.equal(a.cpu(), b), i
        run(step.to(DEV), *state())  # eager work on its own workspace in between
    assert torch.equal(st[3].cpu(), eager[3].cpu())
    assert torch.equal(st[0].cpu(), eager[0].cpu()) and torch.equal(st[1].cpu(), eager[1].cpu())


def test_calls_repeat_bit_for_bit_and_on_other_streams():
    from mtp_hip import ops
    g = gen(14)
    B, H, Hk, D, L, page, T = 1, 8, 2, 128, 9000, 16, 3
    kp, vp, table, _ = make_pages(g, L // page + 2, B, Hk, page, D, L, BF16)
    kd, vd, td = kp.to(DEV), vp.to(DEV), table.to(DEV)
    q = randn(g, B, H, T, D, dtype=BF16).to(DEV)

    def call():
        w = torch.zeros(B, Hk, L, device=DEV)
        return ops.paged_window_attention(q, kd, vd, td, page, L - T, weights=w), w

    first = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:  # two calls at once, each stream with its own workspace
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    for out, w in got:
        assert torch.equal(out, first[0]) and torch.equal(w, first[1])


# ---------------------------------------------------------------------------
# calls at the edges of what the entry points take
@pytest.mark.parametrize("dt,D,rot,inter", [(BF16, 64, 32, False), (F32, 64, 16, True),
                                            (F16, 128, 0, False), (F32, 20, 6, False)])
def test_elements_past_the_rotation_pass_as_they_are(dt, D, rot, inter):
    from mtp_hip import ops
    g = gen(D)
    x = randn(g, 2, 3, 5, D, dtype=dt)
    x[0, 1, 2, rot + 3] = math.inf
    x[1, 2, 4, D - 1] = -math.inf
    x[1, 0, 0, rot] = math.nan
    f = inv_freq(rot).to(DEV)
    for y in ops.qk_norm_rope(x.to(DEV), x.to(DEV), f, 1000, norm=False, interleaved=inter):
        y = y.cpu()
        assert torch.equal(y[..., rot:].nan_to_num(nan=7.0), x[..., rot:].nan_to_num(nan=7.0))
        assert torch.isfinite(y[..., :rot]).all()


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F32, 64), (F16, 24)])
def test_overlapping_and_broadcast_inputs(dt, D):
    """Sliding views (token stride 1, like the elements') and one key head for all."""
    from mtp_hip import ops
    g = gen(21)
    B, H, Hk, T = 2, 4, 2, 9
    q = randn(g, B, H, T + D - 1, dtype=dt).to(DEV).unfold(2, D, 1)
    k = randn(g, B, 1, T, D, dtype=dt).to(DEV).expand(B, Hk, T, D)
    assert q.stride()[2:] == (1, 1) and k.stride(1) == 0
    f = inv_freq(D).to(DEV)
    pos = torch.arange(T).expand(B, T)
    qo, ko = ops.qk_norm_rope(q, k, f)
    for y, x in ((qo, q), (ko, k)):
        ref, mag = S.norm_rotate(x, None, pos, inv_freq(D))
        within(y, ref, rope_bound(ref, mag, dt))
    out = ops.window_attention(q, k, k, 4, 1)
    see = S.visible([0] * B, [T] * B, T, T, 4, 1)
    attn_check(out, q, k, k, see, dt)
    kp, vp, table, _ = make_pages(g, 4, B, Hk, 16, D, 40, dt)
    out = ops.paged_window_attention(q, kp.to(DEV), vp.to(DEV), table.to(DEV), 16, 30)
    see = S.visible([30] * B, [T] * B, T, 40, None, 0)
    attn_check(out, q, S.rows_of(kp, table, 16)[0], S.rows_of(vp, table, 16)[0], see, dt)


@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64)])
def test_window_attention_scales_not_above_zero(dt, D, scale):
    from mtp_hip import ops
    g = gen(22)
    q, k, v = (randn(g, 1, 2, n, D, dtype=dt) for n in (200, 260, 260))
    out = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), 100, 2, scale=scale)
    see = S.visible([60], [200], 200, 260, 100, 2)
    ref, spread, _, _ = S.attention(q, k, v, see, scale=scale)
    score = S.attention(q, k, v, see, scale=abs(scale))[3]
    e = (D + 6) * U * score[..., None]
    h16 = half(dt) if dt is not F32 else 0.0
    within(out, ref, half(dt) * ref.abs() + (h16 + 2 * e + 272 * U) * spread + 2.0 ** -25)


@pytest.mark.parametrize("dt,B,T,L,H,Hk,D,window,sinks", [
    (BF16, 1, 7, 30, 2, 2, 128, None, 0), (BF16, 3, 20, 20, 4, 4, 64, 5, 1),
    (F16, 1, 128, 128, 1, 1, 128, None, 0), (BF16, 2, 65, 64 + 65, 2, 1, 64, 64, 0),
    (F16, 1, 33, 2000, 1, 1, 128, None, 0), (F16, 1, 81, 4091, 4, 2, 64, None, 0),
    (BF16, 1, 33, 9000, 1, 1, 64, None, 0), (BF16, 1, 40, 3000, 2, 1, 128, 900, 5),
    (F32, 1, 40, 1500, 1, 1, 64, None, 0), (F32, 1, 9, 700, 2, 1, 128, 300, 1),
    (BF16, 1, 1, 3000, 2, 1, 64, None, 0)])
def test_few_rows_of_a_prompt(dt, B, T, L, H, Hk, D, window, sinks):
    """Short prompts, and a few rows behind many keys: their keys in chunks."""
    from mtp_hip import ops
    g = gen(T + L)
    q, k, v = (randn(g, B, h, n, D, dtype=dt) for h, n in ((H, T), (Hk, L), (Hk, L)))
    print(f"case rows {dt} {(B, T, L, H, Hk, D, window, sinks)}", flush=True)
    args = [x.to(DEV) for x in (q, k, v)]
    see = S.visible([L - T] * B, [T] * B, T, L, window, sinks)
    out = ops.window_attention(*args, window, sinks)
    attn_check(out, q, k, v, see, dt)
    assert torch.equal(out, ops.window_attention(*args, window, sinks))
    # a NaN value that the first row alone does not see
    if window is None and T > 1:
        v[:, :, L - T + 1, 3] = math.nan
        out = ops.window_attention(args[0], args[1], v.to(DEV)).cpu()
        assert torch.isnan(out[:, :, 1:, 3]).all() and torch.isfinite(out[:, :, 0]).all()


@pytest.mark.parametrize("L,keep", [(4096, 64), (4097, 300), (9000, 65), (20000, 64), (33000, 100)])
def test_kv_evict_lengths(L, keep):
    """Entries of a thread in registers (up to 4, 8, 16, 32 of them) or not, and
    rows moved by the selecting workgroup."""
    from mtp_hip import ops
    g = gen(L)
    B, Hk, D, page = 2, 1, 64, 64
    P = L // page + keep // page + 4
    w = torch.randint(0, 200, (B, Hk, L), generator=g).float()
    kp, vp, table, out_table = make_pages(g, P, B, Hk, page, D, L, BF16, keep)
    kd, vd = kp.to(DEV), vp.to(DEV)
    n = [L, L // 2 + 3]
    got = ops.kv_evict(w.to(DEV), torch.tensor(n).to(DEV), kd, vd, table.to(DEV),
                       out_table.to(DEV), 4, 20)
    want = S.evict(w, n, kp, vp, table, out_table, 4, 20)
    for a, b in zip(got + (kd, vd), want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_pages_past_32_bits(dt):
    """A pool of more than 2^31 elements, read and written at its far end: the
    same results as from a small one."""
    from mtp_hip import ops
    g = gen(24)
    B, H, Hk, D, page, L, T, keep = 1, 4, 1, 128, 16, 300, 5, 60
    small = 64
    kp, vp, table, out_table = make_pages(g, small, B, Hk, page, D, L, dt, keep)
    P = 2 ** 31 // (Hk * page * D) + small
    big = [torch.empty(P, B, Hk, page, D, dtype=dt, device=DEV) for _ in range(2)]
    for to, x in zip(big, (kp, vp)):
        to[P - small:] = x.to(DEV)
    q, k, v = (randn(g, B, h, T, D, dtype=dt).to(DEV) for h in (H, Hk, Hk))
    f = inv_freq(D).to(DEV)
    runs = []
    for (kd, vd), base in (((kp.to(DEV), vp.to(DEV)), 0), (big, P - small)):
        td, od = (x.to(DEV) + base for x in (table, out_table))
        w = torch.zeros(B, Hk, L, device=DEV)
        qr = ops.qk_norm_rope_write(q, k, v, f, kd, vd, td, L - T)
        out = ops.paged_window_attention(qr, kd, vd, td, page, L - T, weights=w)
        cut = ops.kv_evict(w, torch.tensor([L]).to(DEV), kd, vd, td, od, 1, 8)
        runs.append([x.cpu() for x in (qr, out, w, *cut, kd[base:base + small],
                                       vd[base:base + small])])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_dense_keys_past_32_bits(dt):
    """Key rows so far apart that their offsets pass 2^31 elements."""
    from mtp_hip import ops
    g = gen(25)
    T, L, D, apart = 200, 270, 64, 1 << 23
    q, k, v = (randn(g, 1, 1, n, D, dtype=dt) for n in (T, L, L))
    room = torch.empty((L - 1) * apart + 2 * D, dtype=dt, device=DEV)
    rows = room.as_strided((1, 1, L, 2 * D), (0, 0, apart, 1))
    rows.copy_(torch.cat([k, v], -1).to(DEV))
    out = ops.window_attention(q.to(DEV), rows[..., :D], rows[..., D:], 100, 3)
    see = S.visible([L - T], [T], T, L, 100, 3)
    attn_check(out, q, k, v, see, dt)


@pytest.mark.parametrize("L,n,keep", [(1000, 997, 300), (5003, 5003, 2000), (40003, 40001, 700)])
def test_kv_evict_ties_across_lanes(L, n, keep):
    """Few distinct weights, so that the last ones kept are equals of many that are
    not, in lanes and waves on both sides; rows that start at any word."""
    from mtp_hip import ops
    g = gen(L)
    B, Hk, page = 1, 3, 16
    P = L // page + keep // page + 4
    w = torch.randint(0, 4, (B, Hk, L), generator=g).float()
    kp, vp, table, out_table = make_pages(g, P, B, Hk, page, 4, L, BF16, keep)
    kept, ow, new = ops.kv_evict(w.to(DEV), torch.tensor([n]).to(DEV), kp.to(DEV), vp.to(DEV),
                                 table.to(DEV), out_table.to(DEV), 3, 50)
    key = w[..., :n].double()
    key[..., :3] = key[..., n - 50:] = math.inf
    ref = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    assert torch.equal(kept.cpu().long(), ref) and int(new) == keep
    assert torch.equal(ow.cpu(), torch.gather(w, 2, ref))


@pytest.mark.parametrize("dt,n,T,L,H,Hk,D,window,sinks", [
    (F16, [7000], 500, 7000, 16, 8, 64, None, 0), (BF16, [8000], 260, 8000, 8, 4, 128, None, 0),
    (BF16, [8000, 7601, 5, 7900], 400, 8000, 4, 2, 128, None, 0),
    (F16, [9000, 8999, 0, 8800], 300, 9000, 8, 4, 64, 8500, 40)])
def test_chunk_behind_many_keys(dt, n, T, L, H, Hk, D, window, sinks):
    """Some hundred rows behind thousands of keys (few blocks, their keys in chunks),
    ragged with garbage behind, and a value that only some rows see."""
    from mtp_hip import ops
    g = gen(T + L)
    B = len(n)
    print(f"case chunk {dt} {(n, T, L, H, Hk, D, window, sinks)}", flush=True)
    q, k, v = (randn(g, B, h, m, D, dtype=dt) for h, m in ((H, T), (Hk, L), (Hk, L)))
    for b in range(B):
        k[b, :, n[b]:] = math.nan
        v[b, :, n[b]:] = math.inf
        q[b, :, max(0, n[b] - (L - T)):] = math.nan
    dev = [x.to(DEV) for x in (q, k, v)]
    lengths = torch.tensor(n).to(DEV) if B > 1 else None
    out = ops.window_attention(*dev, window, sinks, lengths=lengths)
    see = S.visible([L - T] * B, [max(0, e - (L - T)) for e in n], T, L, window, sinks)
    attn_check(out, q.nan_to_num(), k.nan_to_num(), v.nan_to_num(posinf=0.0), see, dt)
    assert torch.equal(out, ops.window_attention(*dev, window, sinks, lengths=lengths))
    dev[2][0, :, L - T + 10, 2] = math.nan
    bad = ops.window_attention(*dev, window, sinks, lengths=lengths)
    assert torch.isnan(bad[0, :, 10:, 2]).all()
    assert torch.equal(bad[0, :, :10], out[0, :, :10]) or \
        torch.isfinite(bad[0, :, :10]).all()
    assert torch.equal(bad[1:], out[1:])


def test_chunks_captured_and_replayed():
    """Keys in chunks and their join as a graph, replayed among eager calls."""
    from mtp_hip import ops
    g = gen(31)
    q, k, v = (randn(g, 1, h, m, 64, dtype=BF16).to(DEV) for h, m in ((8, 300), (4, 9000), (4, 9000)))
    want = [ops.window_attention(q * s, k, v).clone() for s in (1, 2, 3)]
    x = q.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.window_attention(x, k, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = ops.window_attention(x, k, v)
    for s in (1, 2, 3):
        x.copy_(q * s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[s - 1])
        ops.window_attention(q, k, v)
        torch.cuda.synchronize()
