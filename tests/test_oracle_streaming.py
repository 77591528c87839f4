"""Pins of oracle/streaming.py, and the host side of the streaming ops: plans, cache layout, refusals."""
import numpy as np
import pytest
import torch

from oracle import attention as OA
from oracle import rope as OR
from oracle import streaming as O
from qvggt_amd import awq_inference_engine as E
from qvggt_amd.kv_cache import Int8KVCache


# ------------------------------------------------------------------- oracle
def test_rope_axes_quarter_turn_and_copy():
    """One pair of one axis at 2 pi / 4 radians a position: position 1 maps (a, b) to (-b, a)."""
    x = np.array([[[3.0, 5.0, 7.0, 9.0]]] * 2)
    y = O.rope_axes(x, [[0], [1]], [(0, 1, 0, np.pi / 2)])
    assert np.array_equal(y[0], x[0])
    np.testing.assert_allclose(y[1, 0], [-5, 3, 7, 9], atol=1e-14)


def test_rope_axes_block_layout_is_rope2d():
    T, H = 50, 3
    rng = np.random.default_rng(0)
    x = rng.standard_normal((T, H, 64)).astype(np.float16)
    pos = rng.integers(0, 38, (T, 2)).astype(np.int32)
    want = np.asarray(OR.rope2d(x, pos, *OR.rope2d_tables(38)), np.float64)
    np.testing.assert_allclose(O.rope_axes(x, pos, O.rope_pairs((32, 32), "block")), want, atol=4e-3)   # want is fp16


def test_rope_pairs_half_layout():
    p = O.rope_pairs((4, 2), "half", 10.0)
    assert [t[:3] for t in p] == [(0, 3, 0), (1, 4, 0), (2, 5, 1)]
    assert [t[3] for t in p] == [1.0, 10.0 ** (-2 / 6), 10.0 ** (-4 / 6)]


@pytest.mark.parametrize("amax,scale", [(127.0, 1.0), (126.0, 1.0), (127.1, 1.125), (1.0, 9 / 1024),
                                        (65504.0, 576.0), (0.0, 0.0), (2.0 ** -24, 9 * 2.0 ** -34), (1e-37, 2.0 ** -120)])
def test_scale_by_hand(amax, scale):
    """127 -> 1; 127.1 -> the next number of four bits, 1.125; 1/127 = 8.06 / 1024 ->
    9 / 1024; 65504 / 127 = 515.8 -> 1.125 * 512."""
    assert O.scale_of(amax) == scale


def test_cache_codes_by_hand():
    c = O.Cache(128, 1, 2)
    c.append(np.array([[[127.0, -0.5]], [[1.5, 2.5]]]))            # scale 1, ties to even
    assert c.scales[0, 0] == 1 and c.codes[:2, 0].tolist() == [[127, 0], [2, 2]]
    c.append(np.array([[[250.0, -4.0]]]))                          # 250 / 127 = 1.97 -> 2: codes halve
    assert c.scales[0, 0] == 2 and c.codes[:3, 0].tolist() == [[64, 0], [1, 1], [125, -2]]
    c.append(np.array([[[4.0, 0.0]]]))                             # the scale stays
    assert c.scales[0, 0] == 2 and c.codes[3, 0].tolist() == [2, 0] and c.len == 4
    c.append(np.zeros((0, 1, 2)), start=3)
    assert c.len == 3 and c.values().tolist()[2] == [[250, -4]]


def test_attention_agrees_with_the_square_one():
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((20, 2, 64)) for _ in range(3))
    np.testing.assert_allclose(O.attention(q, k, v, 0.125), OA.attention_ref(q, k, v, 1, 20), atol=1e-12)
    keep = np.zeros(20, bool)
    keep[[3, 7]] = True
    np.testing.assert_allclose(O.attention(q, k, v, 0.125, keep),
                               O.attention(q, k[[3, 7]], v[[3, 7]], 0.125), atol=1e-12)
    assert not O.attention(q, k, v, 0.125, np.zeros(20, bool)).any()
    v[4] = np.nan                                                  # not kept, not read
    assert np.isfinite(O.attention(q, k, v, 0.125, keep)).all()
    shared = O.attention(np.repeat(q, 2, 1), k, v[:, :], 0.125, keep)
    np.testing.assert_array_equal(shared[:, 0], O.attention(q, k, v, 0.125, keep)[:, 0])


# ------------------------------------------------------------------ host side
def test_rope_axes_plan():
    p = E.rope_axes_plan(64, (16, 24, 20), base=50.0)
    want = [t[3] / (2 * np.pi) for t in O.rope_pairs((16, 24, 20), "block", 50.0)]
    assert p.turns[:30].tolist() == pytest.approx(want, rel=1e-15) and p.turns[30:].tolist() == [0, 0]
    f = E.rope_axes_plan(64, (32,), frequencies=np.arange(16.0), layout="half")
    assert f.turns[:16].tolist() == pytest.approx((np.arange(16) / (2 * np.pi)).tolist(), rel=1e-15)
    for bad in (dict(head_dim=64, sections=(15, 3)), dict(head_dim=64, sections=(64, 2)), dict(head_dim=64, sections=()),
                dict(head_dim=64, sections=(2,) * 5), dict(head_dim=63, sections=(2,)), dict(head_dim=64, sections=(0, 2)),
                dict(head_dim=64, sections=(4,), layout="x"), dict(head_dim=64, sections=(4,), frequencies=[1.0]),
                dict(head_dim=64, sections=(4,), frequencies=[1.0, float("nan")])):
        with pytest.raises(RuntimeError, match="rope_axes_plan"):
            E.rope_axes_plan(**bad)


def test_rope_axes_refusals():
    plan = E.rope_axes_plan(64, (32, 32))
    x = torch.zeros(5, 3, 64, dtype=torch.float16)
    pos = torch.zeros(5, 2, dtype=torch.int32)
    for args, msg in (((x[..., :32], pos, plan), "x must be"), ((x[0], pos, plan), "x must be"),
                      ((x.double(), pos, plan), "unsupported dtype"), ((x, pos.long(), plan), "positions must be"),
                      ((x, pos[:4], plan), "positions must be"), ((x, pos[:, :1], plan), "positions must be"),
                      ((x, pos, plan.turns), "plan must come"), ((x, pos, plan, x.float()), "out must be"),
                      ((x, pos, plan, torch.zeros(5, 1, 64).half().expand(5, 3, 64)), "overlap itself"),
                      ((x, pos, plan, torch.zeros(5, 3, 128).half()[..., ::2]), "unit dim stride"),
                      ((x[:, :2], pos, plan, x.view(-1)[:640].view(5, 2, 64)), "in place"),
                      ((x, pos, plan._replace(turns=plan.turns.float())), "turns"),
                      ((x, pos, plan), "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            E.rope_axes(*args)


def test_rope_axes_in_place_of_one_or_no_token():
    """The stride of a dim of one or none says nothing: a view of the same token, empty tensors of any strides are taken."""
    plan = E.rope_axes_plan(64, (32, 32))
    qkv = torch.zeros(4, 9, 64, dtype=torch.float16)
    one = qkv[:1, :3]
    for x, out in ((one, qkv.view(-1)[:192].view(1, 3, 64)),
                   (qkv[:, :1][:1], qkv.view(-1)[:64].view(1, 1, 64)), (qkv[:0, :3], torch.empty(0, 3, 64, dtype=torch.float16))):
        assert x.data_ptr() == out.data_ptr() and x.stride() != out.stride()
        with pytest.raises(RuntimeError, match="GPU only"):
            E.rope_axes(x, torch.zeros(len(x), 2, dtype=torch.int32), plan, out)
    with pytest.raises(RuntimeError, match="in place"):
        E.rope_axes(qkv[:2, :3], torch.zeros(2, 2, dtype=torch.int32), plan, qkv.view(-1)[:384].view(2, 3, 64))


def test_cache_refusals():
    for bad in (dict(batch=0, kv_heads=1, head_dim=64, capacity=1), dict(batch=1, kv_heads=0, head_dim=64, capacity=1),
                dict(batch=1, kv_heads=1, head_dim=96, capacity=1), dict(batch=1, kv_heads=1, head_dim=64, capacity=0)):
        with pytest.raises(RuntimeError, match="Int8KVCache"):
            Int8KVCache(**bad, device="cpu")
    c = Int8KVCache(2, 3, 64, 100, device="cpu")
    assert c.capacity == 128 and c.blocks == 2
    k = torch.zeros(2, 5, 3, 64, dtype=torch.float16)
    one = torch.zeros(2, dtype=torch.int32)
    for args, kw, msg in (((k, k[:, :4]), {}, "v must be"), ((k.float(), k), {}, "data type"), ((k, k.bfloat16()), {}, "v must be"),
                          ((k[:1], k[:1]), {}, "k must be"), ((k[..., :32], k), {}, "k must be"),
                          ((torch.zeros(2, 129, 3, 64).half(),) * 2, {}, "do not fit"),
                          ((k, k), dict(counts=one.long()), "counts must be"), ((k, k), dict(start=one[:1]), "start must be"),
                          ((k, k), dict(start=torch.zeros(2, 2, dtype=torch.int32)[:, 0]), "contiguous"),
                          ((k, k), {}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            c.append(*args, **kw)
    for kw, msg in ((dict(n=-1), "number of tokens"), (dict(dtype=torch.int8), "dtype"), (dict(first=one.float()), "first must"),
                    ({}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            c.values(**kw)


def test_cache_limits_are_those_of_the_c_entries():
    """The largest capacity and range pass both sides; one block or token more is refused before anything is allocated."""
    from qvggt_amd import _lib
    most = (1 << 29) - 64
    c = Int8KVCache(1, 1, 64, most, device="meta")
    assert c.capacity == most and c.blocks == (1 << 23) - 1
    for capacity in (most + 1, 1 << 29):
        with pytest.raises(RuntimeError, match="bad batch"):
            Int8KVCache(1, 1, 64, capacity, device="meta")
    with pytest.raises(RuntimeError, match="number of tokens"):
        c.values(1 << 29)
    with pytest.raises(RuntimeError, match="GPU only"):
        c.values((1 << 29) - 1)
    lib, p = _lib.load(), 1 << 20
    val = lambda n, blocks: lib.qv_kv8_values(p, p, p, p, p, None, None, p, 2, 1, n, 1, 64, blocks, None)
    said = lambda: lib.qv_last_error().decode()
    assert val(5, 1 << 23) == -1 and "cache shape" in said() and val(1 << 29, 3) == -1 and "number of tokens" in said()
    # what Python lets through comes to the next check, the null output
    assert val((1 << 29) - 1, c.blocks) == -1 and "null" in said()


def test_cross_split_of_many_heads():
    """One query, 128 to 255 heads: no split while the keys and values stay in the caches (256 MB), two behind that;
    from a head for each CU on never."""
    part = lambda heads, D: heads * (4 * D + 8)
    need = lambda heads, D, keys: E._kv_workspace_bytes(0, heads, 1, 1, 1, D, keys)
    for D in (64, 128):
        fits = (256 << 20) // (4 * 128 * D)
        assert need(128, D, 1374) == need(128, D, fits) == need(256, D, 40000) == 0
        assert need(128, D, fits + 1) == need(128, D, 43968) == 2 * part(128, D)
        assert need(120, D, 1374) == 2 * part(120, D)


@pytest.mark.parametrize("D", [64, 128])
def test_cache_block_order_is_a_permutation(D):
    key, val = Int8KVCache(1, 1, D, 64, device="cpu")._order()
    for o in (key, val):
        assert o.shape == (64, D) and torch.equal(o.reshape(-1).sort()[0], torch.arange(64 * D))
    # a lane's unit: 16 dims of one token; the 16 tokens of one dim that its registers meet
    assert (key.view(64, D // 16, 16).diff(dim=2) == 1).all()
    toks = torch.empty(64 * D, dtype=torch.long)
    toks[val.reshape(-1)] = torch.arange(64 * D) // D
    assert toks[:16].tolist() == [0, 1, 2, 3, 8, 9, 10, 11, 16, 17, 18, 19, 24, 25, 26, 27]
    assert toks[32 * 16:33 * 16].tolist() == [4, 5, 6, 7, 12, 13, 14, 15, 20, 21, 22, 23, 28, 29, 30, 31]


def test_attention_kv_refusals():
    q, k = torch.zeros(2, 5, 4, 64, dtype=torch.float16), torch.zeros(2, 9, 2, 64, dtype=torch.float16)
    lens, mask = torch.zeros(2, dtype=torch.int32), torch.ones(2, 9, dtype=torch.bool)
    for args, kw, msg in (((q, k, k[:, :8]), {}, "k and v must be"), ((q[0], k, k), {}, "q must be"),
                          ((q.float(), k, k), {}, "data type"), ((q, k.bfloat16(), k), {}, "k and v must be"),
                          ((q[:, :, :3], k, k), {}, "not a multiple"), ((q[..., :32], k, k), {}, "q must be"),
                          ((q[:1], k, k), {}, "k must be"), ((q, k, k), dict(scale=0.0), "scale"),
                          ((q, k, k), dict(scale=float("nan")), "scale"), ((q, k, k), dict(scale=-1.0), "scale"),
                          ((q, k, k), dict(kv_lens=lens.long()), "kv_lens"), ((q, k, k), dict(kv_lens=lens[:1]), "kv_lens"),
                          ((q, k, k), dict(key_mask=mask.int()), "key_mask"), ((q, k, k), dict(key_mask=mask[:, :8]), "key_mask"),
                          ((q, k, k), dict(out=q.float()), "out must be"), ((q, k, k), dict(out=q[:, :4]), "out must be"),
                          ((q, k, k), dict(out=q[:, :1].expand(2, 5, 4, 64)), "out must be"),
                          ((q, k, k), dict(out=torch.zeros(2, 5, 4, 66).half()[..., 1:65]), "8-byte"),
                          ((q, k, k), {}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            E.cross_attention(*args, **kw)
    c = Int8KVCache(2, 2, 64, 100, device="cpu")
    for args, kw, msg in (((q[:1],), {}, "q must be"), ((torch.zeros(2, 5, 4, 128).half(),), {}, "q must be"),
                          ((q[:, :, :3],), {}, "not a multiple"), ((q,), dict(counts=lens.long()), "counts"),
                          ((q,), dict(scale=float("inf")), "scale"), ((q,), dict(out=q[:, :2]), "out must be"),
                          ((q,), {}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            c.attention(*args, **kw)


def test_cache_length_hint(monkeypatch):
    """How many keys the attention's split is laid out for: the tokens appended so far, the capacity once a start was
    given (it lies on the GPU and may be anything), or what the caller says.  No kernel runs here."""
    import contextlib

    from qvggt_amd import kv_cache as M
    calls = []
    monkeypatch.setattr(M, "_on_gpu", lambda *t, what: 0)
    monkeypatch.setattr(M, "_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(M, "_stream", lambda dev: 0)
    monkeypatch.setattr(M._lib, "call", lambda name, *args: calls.append((name, args)))
    c = Int8KVCache(1, 1, 64, 1 << 20, device="cpu")
    q, k = torch.zeros(1, 1, 4, 64).half(), torch.zeros(1, 100, 1, 64).half()
    at = torch.tensor([(1 << 20) - 100], dtype=torch.int32)

    def keys(**kw):
        c.attention(q, **kw)
        name, args = calls[-1]
        assert name == "qv_kv8_attention"
        assert args[-2] == E._kv_workspace_bytes(1, 1, 1, 4, 1, 64, args[16])     # the workspace of the same plan
        return args[16]

    assert keys() == 0 and keys(longest=5000) == 5000
    c.append(k, k)
    assert keys() == 100 and keys(longest=0) == 0 and keys(longest=1 << 30) == 1 << 20
    c.append(k, k, start=c.lens)                           # its own lengths
    assert keys() == 200
    c.append(k, k, start=at)                               # far behind them: one split would walk 16384 blocks
    assert keys() == 1 << 20
    c.reset()
    assert keys() == 0
    c.append(k, k)
    for _ in range(5):                                     # back and forth: not 100 more each time
        c.append(k, k, start=at)
        assert keys() == 1 << 20 and keys(longest=300) == 300
    with pytest.raises(RuntimeError, match="longest"):
        c.attention(q, longest=-1)


def test_c_entries_refuse():
    """Bad arguments end at the C entries with a message, before any device work (pointers here are never followed)."""
    import ctypes as C

    from qvggt_amd import _lib
    lib = _lib.load()
    st = (C.c_int64 * 3)(64 * 8, 64, 64)
    odd = (C.c_int64 * 3)(64 * 8, 60, 64)
    p = 1 << 20

    def refused(rc, what):
        assert rc == -1 and what in lib.qv_last_error().decode(), (rc, lib.qv_last_error())

    rope = lambda **kw: lib.qv_rope_axes(*{**dict(x=p, out=p, dt=0, pos=p, turns=p, sec=(C.c_int64 * 2)(32, 32), axes=2, layout=0,
                                                  T=5, H=2, D=64, a=128, b=64, c=128, d=64, s=None), **kw}.values())
    for kw, what in ((dict(dt=7), "dtype"), (dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(layout=2), "layout"),
                     (dict(D=63), "shape"), (dict(H=5000), "shape"), (dict(sec=(C.c_int64 * 2)(31, 2)), "section"),
                     (dict(sec=(C.c_int64 * 2)(64, 2)), "sections"), (dict(x=None), "null"), (dict(turns=None), "null"),
                     (dict(x=p + 1), "aligned")):
        refused(rope(**kw), what)
    assert rope(T=0) == 0
    app = lambda **kw: lib.qv_kv8_append(*{**dict(k=p, v=p, dt=0, kc=p, vc=p, ks=p, vs=p, start=p, lens=p, tick=p, counts=None, B=1,
                                                  n=5, Hk=2, D=64, blocks=3, kst=st, vst=st, s=None), **kw}.values())
    for kw, what in ((dict(D=32), "head_dim"), (dict(n=193), "do not fit"), (dict(dt=2), "dtype"), (dict(kst=odd), "strides"),
                     (dict(k=p + 2), "aligned"), (dict(kc=p + 8), "aligned"), (dict(lens=None), "null"), (dict(blocks=0), "cache shape"),
                     (dict(B=40000), "cache shape"), (dict(blocks=1 << 24), "cache shape"), (dict(k=None), "null")):
        refused(app(**kw), what)
    assert app(B=0) == 0
    val = lambda **kw: lib.qv_kv8_values(*{**dict(kc=p, vc=p, ks=p, vs=p, lens=p, first=None, ko=p, vo=p, dt=2, B=1, n=5, Hk=2, D=64,
                                                  blocks=3, s=None), **kw}.values())
    for kw, what in ((dict(dt=3), "dtype"), (dict(n=-1), "number of tokens"), (dict(ko=None), "null"), (dict(vo=p + 4), "aligned")):
        refused(val(**kw), what)
    assert val(n=0) == 0
    cross = lambda **kw: lib.qv_attention_cross(*{**dict(q=p, k=p, v=p, out=p, dt=0, lens=None, mask=None, ms=0, B=1, Lq=5, Lk=9, H=4,
                                                         Hk=2, D=64, qs=st, ks=st, vs=st, os=st, scale=0.1, ws=None, wb=0, s=None),
                                                  **kw}.values())
    far = (C.c_int64 * 3)(64, 1 << 25, 64)
    for kw, what in ((dict(dt=2), "dtype"), (dict(D=96), "head_dim"), (dict(Hk=3), "shape"), (dict(scale=0.0), "scale"),
                     (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(q=p + 8), "aligned"),
                     (dict(k=p + 8), "aligned"), (dict(qs=odd), "strides"), (dict(ks=odd), "strides"), (dict(vs=far), "token strides"),
                     (dict(ks=(C.c_int64 * 3)(64, 0, 64)), "token strides"), (dict(v=None), "null"), (dict(out=None), "null"),
                     (dict(B=70000), "grid"), (dict(Lq=1 << 27, H=256, Hk=2), "rows")):
        refused(cross(**kw), what)
    assert cross(B=0) == 0 and cross(Lq=0) == 0
    att = lambda **kw: lib.qv_kv8_attention(*{**dict(q=p, out=p, dt=0, kc=p, vc=p, ks=p, vs=p, lens=p, counts=None, causal=0, B=1,
                                                     Lq=5, H=4, Hk=2, D=64, blocks=3, keys=100, qs=st, os=st, scale=0.1, ws=None,
                                                     wb=0, s=None), **kw}.values())
    for kw, what in ((dict(blocks=0), "blocks"), (dict(lens=None), "null"), (dict(kc=p + 8), "aligned"), (dict(D=32), "head_dim"),
                     (dict(scale=-1.0), "scale"), (dict(H=5), "shape")):
        refused(att(**kw), what)
    need = lib.qv_attention_kv_workspace
    assert need(1, 1, 1, 8, 1, 96, 5000) == 0 and need(1, 1, 1, 8, 3, 64, 5000) == 0 and need(1, 0, 1, 8, 1, 64, 5000) == 0
    assert need(1, 1, 1, 8, 1, 64, 64) == 0 and need(0, 1, 1, 8, 1, 64, 100000) > 0
