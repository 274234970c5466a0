"""What the serving operators refuse (CPU): shapes, types, options and host
tensors in Python before any library call, and sizes, null pointers and types
in the C ABI before any HIP call; and the oracle against brute force."""
import math
import os

import pytest
import torch

from mtp_hip import _lib, ops
from oracle import serving as S

B, H, Hk, T, D, L, PS, P = 2, 4, 2, 3, 8, 32, 4, 20


def tensors(dt=torch.float32):
    q = torch.randn(B, H, T, D).to(dt)
    k = torch.randn(B, Hk, T, D).to(dt)
    pages = torch.randn(P, B, Hk, PS, D).to(dt)
    table = torch.zeros(B, L, dtype=torch.int32)
    return q, k, pages, table


FREQ = torch.ones(D // 2)


@pytest.mark.parametrize("change", [
    dict(k=torch.randn(B, Hk, T + 1, D)), dict(k=torch.randn(B, Hk, T, D - 1)),
    dict(k=torch.randn(B, Hk, T, D).bfloat16()), dict(q=torch.randn(B, H, D)),
    dict(f=torch.ones(D // 2 + 1)), dict(f=torch.ones(2, 2)),
    dict(positions=torch.zeros(T + 1, dtype=torch.int64)),
    dict(positions=torch.zeros(B + 1, T, dtype=torch.int64)),
    dict(q_weight=torch.ones(D + 1)), dict(k_weight=torch.ones(1)),
    dict(start=torch.zeros(B + 1, dtype=torch.int64)),
])
def test_qk_norm_rope_shapes(change):
    q, k, _, _ = tensors()
    a = dict(q=q, k=k, f=FREQ, start=0, positions=None, q_weight=None, k_weight=None)
    a.update(change)
    with pytest.raises(AssertionError):
        ops.qk_norm_rope(a["q"], a["k"], a["f"], a["start"], a["positions"], a["q_weight"],
                         a["k_weight"])


def test_types_and_host_tensors():
    q, k, pages, table = tensors()
    with pytest.raises(TypeError, match="float32 or float64"):
        ops.qk_norm_rope(q, k, FREQ.bfloat16())
    for call in (lambda: ops.qk_norm_rope(q, k, FREQ),
                 lambda: ops.qk_norm_rope_write(q, k, k, FREQ, pages, pages, table, 0),
                 lambda: ops.window_attention(q, k, k),
                 lambda: ops.paged_window_attention(q, pages, pages, table, PS, 0),
                 lambda: ops.kv_evict(torch.zeros(B, Hk, L), torch.zeros(B), pages, pages, table,
                                      torch.ones(B, 5, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def test_write_and_paged_shapes():
    q, k, pages, table = tensors()
    for bad in (pages[:, :1], pages[..., :4], pages.transpose(2, 3), pages.bfloat16(), pages[0]):
        with pytest.raises(AssertionError):
            ops.qk_norm_rope_write(q, k, k, FREQ, bad, bad, table, 0)
        with pytest.raises(AssertionError):
            ops.paged_window_attention(q, bad, bad, table, PS, 0)
    with pytest.raises(AssertionError):
        ops.qk_norm_rope_write(q, k, k[:, :1], FREQ, pages, pages, table, 0)
    with pytest.raises(AssertionError):
        ops.qk_norm_rope_write(q, k, k, FREQ, pages, pages, table[:1], 0)
    for kw in (dict(page_size=PS + 1), dict(page_table=table[0]), dict(q=q[:, :3]),
               dict(start=torch.zeros(3)), dict(weights=torch.zeros(B, Hk, L + 1)),
               dict(weights=torch.zeros(B, Hk, L).double()),
               dict(weights=torch.zeros(B, L, Hk).transpose(1, 2))):
        a = dict(q=q, page_table=table, page_size=PS, start=0, weights=None)
        a.update(kw)
        with pytest.raises(AssertionError):
            ops.paged_window_attention(a["q"], pages, pages, a["page_table"], a["page_size"],
                                       a["start"], weights=a["weights"])


def test_window_attention_arguments():
    q, k, _, _ = tensors()
    for kk, vv in ((k[:, :, :2], k[:, :, :2]), (k, k[:1]), (k[:1], k[:1]), (k[..., :4], k[..., :4]),
                   (k.bfloat16(), k.bfloat16()), (k, k.bfloat16())):
        with pytest.raises(AssertionError):
            ops.window_attention(q, kk, vv)
    with pytest.raises(AssertionError):
        ops.window_attention(q[:, :3], k, k)
    with pytest.raises(AssertionError):
        ops.window_attention(q, k, k, lengths=torch.zeros(B + 1, dtype=torch.int64))
    for w, s in ((0, 0), (-1, 0), (4, -1)):
        with pytest.raises(ValueError):
            ops.window_attention(q, k, k, w, s)


def test_kv_evict_arguments():
    _, _, pages, table = tensors()
    w, n = torch.zeros(B, Hk, L), torch.zeros(B, dtype=torch.int64)
    out = torch.ones(B, 6, dtype=torch.int32)
    for kw in (dict(w=w.double()), dict(w=w[:, :1]), dict(w=w[..., :5]), dict(n=n[:1]),
               dict(out=out[:1]), dict(out=out[:, :0]), dict(table=table[:, :5])):
        a = dict(w=w, n=n, table=table, out=out)
        a.update(kw)
        with pytest.raises(AssertionError):
            ops.kv_evict(a["w"], a["n"], pages, pages, a["table"], a["out"])
    for s, r in ((-1, 0), (0, -1), (3, 4), (7, 0)):
        with pytest.raises(ValueError):
            ops.kv_evict(w, n, pages, pages, table, out, s, r)
    with pytest.raises(ValueError, match="onto themselves"):
        ops.kv_evict(w, n, pages, pages, table, table)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.fail("libmtp_hip.so not built: run python mtp-engine_amd/build.py")
    return _lib.load()


X = 4096  # never dereferenced: every call below returns before any HIP call
STR = (64, 64, 64)


def rope_pack(q=X, k=X, v=X, qo=X, ko=X, kp=X, vp=X, tab=X, f=X, b=1, t=2, h=2, hk=1, d=64, rot=64,
              np_=4, ps=16, ld=8, dt=_lib.BF16):
    z = [x or 0 for x in (q, k, v, qo, ko, kp, vp, tab, f)]
    return _lib.ROPE_ARGS.pack(*z, 0, 0, 0, 0, b, t, h, hk, d, *STR, *STR, *STR, *STR, *STR, rot, 0,
                               0, np_, ps, ld, 1e-6, dt, 0, 0, 1, 0)


def test_rope_abi(lib):
    for fn, write in ((lib.mtp_qk_norm_rope, False), (lib.mtp_qk_norm_rope_write, True)):
        def call(**kw):
            return fn(rope_pack(**kw), None)
        assert fn(None, None) == _lib.ERR_NULL
        assert call(dt=_lib.FP8E4M3) == _lib.ERR_DTYPE
        for kw in (dict(d=0), dict(d=5000), dict(rot=63), dict(rot=66), dict(rot=-2), dict(b=-1),
                   dict(h=70000)):
            assert call(**kw) == _lib.ERR_SHAPE, kw
        nulls = [dict(q=None), dict(k=None), dict(f=None), dict(qo=None)]
        nulls += [dict(v=None), dict(kp=None), dict(vp=None), dict(tab=None)] if write else \
            [dict(ko=None)]
        for kw in nulls:
            assert call(**kw) == _lib.ERR_NULL, kw
        if write:
            for kw in (dict(np_=-1), dict(ps=0), dict(ld=-1)):
                assert call(**kw) == _lib.ERR_SHAPE, kw
        assert call(b=0, q=None, k=None) == _lib.OK and call(t=0) == _lib.OK


def test_window_attention_abi(lib):
    def pack(q=X, k=X, v=X, o=X, tab=X, weights=None, ws=None, nb=0, b=1, h=2, hk=1, t=2, d=64,
             l_=8, w=-1, s=0, np_=4, ps=16, dt=_lib.BF16):
        z = [x or 0 for x in (q, k, v, o, tab, None, None, weights, ws)]
        return _lib.WINDOW_ARGS.pack(*z, nb, b, h, hk, t, d, l_, *STR, *STR, *STR, *STR, w, s, 0,
                                     np_, ps, 1.0, dt, 0)

    for fn, paged in ((lib.mtp_window_attention, False), (lib.mtp_paged_window_attention, True)):
        def call(**kw):
            return fn(pack(**kw), None)
        assert fn(None, None) == _lib.ERR_NULL
        assert call(dt=_lib.I32) == _lib.ERR_DTYPE
        for kw in (dict(h=3, hk=2), dict(hk=0), dict(d=0), dict(d=1025), dict(l_=1 << 30),
                   dict(b=-1), dict(np_=-1) if paged else dict(t=9),
                   dict(ps=0) if paged else dict(t=-1), dict(l_=-1)):
            assert call(**kw) == _lib.ERR_SHAPE, kw
        for kw in (dict(w=0), dict(w=-2), dict(s=-1)):
            assert call(**kw) == _lib.ERR_ARG, kw
        for kw in (dict(q=None), dict(k=None), dict(v=None), dict(o=None),
                   dict(tab=None) if paged else dict(q=None)):
            assert call(**kw) == _lib.ERR_NULL, kw
        assert call(t=0, l_=0, k=None, v=None) == _lib.OK and call(b=0) == _lib.OK
    # weights keep the scores in the workspace
    need = lib.mtp_window_attention_workspace_bytes(_lib.BF16, 1, 2, 1, 2, 64, 8, -1, 0, 1, 1)
    assert need > 0
    assert lib.mtp_paged_window_attention(pack(weights=X, ws=X, nb=need - 1), None) == \
        _lib.ERR_WORKSPACE
    assert lib.mtp_window_attention_workspace_bytes(_lib.BF16, 0, 2, 1, 2, 64, 8, -1, 0, 1, 1) == 0
    # a window bounds the scores kept, not the table's width
    wide = lib.mtp_window_attention_workspace_bytes(_lib.BF16, 1, 2, 1, 1, 64, 1 << 20, 64, 4, 1, 1)
    assert wide < 1 << 20


def test_kv_evict_abi(lib):
    def call(w=X, n=X, b=1, hk=1, l_=8, keep=4, s=0, r=0, kp=X, np_=4, ps=16, rb=128, tab=X, o=X,
             kept=X):
        return lib.mtp_kv_evict(w, n, b, hk, l_, keep, s, r, kp, X, np_, ps, rb, tab, o, kept, X,
                                X, None)

    for kw in (dict(keep=0), dict(rb=0), dict(ps=0), dict(np_=-1), dict(l_=-1), dict(b=-1)):
        assert call(**kw) == _lib.ERR_SHAPE, kw
    for kw in (dict(s=-1), dict(r=-1), dict(s=3, r=2)):
        assert call(**kw) == _lib.ERR_ARG, kw
    for kw in (dict(w=None), dict(n=None), dict(kp=None), dict(tab=None), dict(o=None),
               dict(kept=None)):
        assert call(**kw) == _lib.ERR_NULL, kw
    assert call(b=0, w=None) == _lib.OK


# ---------------------------------------------------------------------------
def test_oracle_attention_by_brute_force():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, h, 6, 3, generator=g).double() for h in (2, 1, 1))
    see = S.visible([0], [5], 6, 6, 2, 1)
    out, spread, w, _ = S.attention(q, k, v, see)
    total = torch.zeros(6, dtype=torch.float64)
    for h in range(2):
        for t in range(6):
            js = [j for j in range(6) if j <= t and (t - j < 2 or j < 1)] if t < 5 else []
            e = [math.exp(float(q[0, h, t] @ k[0, 0, j]) / math.sqrt(3)) for j in js]
            ref = sum((x / sum(e) * v[0, 0, j] for x, j in zip(e, js)), torch.zeros(3).double())
            assert torch.allclose(out[0, h, t], ref, atol=1e-12)
            for x, j in zip(e, js):
                total[j] += x / sum(e)
    assert torch.allclose(w[0, 0], total, atol=1e-12) and (spread >= out.abs() - 1e-12).all()


def test_oracle_rotation_by_complex_turns():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 1, 2, 8, generator=g)
    pos, f = torch.tensor([[3, 100]]), torch.tensor([1.0, 0.1, 0.01])
    y, _ = S.norm_rotate(x, None, pos, f, norm=False)
    z, _ = S.norm_rotate(x, None, pos, f, norm=False, interleaved=True)
    for t in range(2):
        for i in range(3):
            turn = complex(math.cos(float(pos[0, t]) * float(f[i])),
                           math.sin(float(pos[0, t]) * float(f[i])))
            a = complex(x[0, 0, t, i], x[0, 0, t, i + 3]) * turn
            b = complex(x[0, 0, t, 2 * i], x[0, 0, t, 2 * i + 1]) * turn
            assert abs(complex(y[0, 0, t, i], y[0, 0, t, i + 3]) - a) < 1e-9
            assert abs(complex(z[0, 0, t, 2 * i], z[0, 0, t, 2 * i + 1]) - b) < 1e-9
        assert torch.equal(y[0, 0, t, 6:], x[0, 0, t, 6:].double())


def test_kv_evict_refuses_its_own_table_in_any_type():
    _, _, pages, table = tensors()
    w, n = torch.zeros(B, Hk, L), torch.zeros(B, dtype=torch.int64)
    long = table.long()
    for t, out in ((long, long), (table, table[:, :6]), (long, long[:, :6])):
        with pytest.raises(ValueError, match="onto themselves"):
            ops.kv_evict(w, n, pages, pages, t, out)
