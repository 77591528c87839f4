"""CPU: the oracle of packed sequences and the paged cache pinned, plans, and what the ops and C entries refuse."""
import contextlib
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged as P
from oracle.streaming import attention
from qvggt_amd import _lib
from qvggt_amd import awq_inference_engine as E
from qvggt_amd.kv_cache import PagedKVCache


def test_packed_and_received_against_plain_attention():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((7, 4, 8)), rng.standard_normal((7, 2, 8)), rng.standard_normal((7, 2, 8))
    got = P.packed(q, k, v, (3, 0, 4), 0.5, 2)
    keep = np.array([[1, 1, 0, 0], [1, 1, 0, 0], [1, 1, 1, 1], [1, 1, 1, 1]], bool)
    np.testing.assert_allclose(got[3:], attention(q[3:], k[3:], v[3:], 0.5, keep), rtol=1e-13)
    np.testing.assert_allclose(got[:3], attention(q[:3], k[:3], v[:3], 0.5, keep[:3, :3]), rtol=1e-13)
    # the values' own weights: attention to one-hot values
    w = P.received(q[3:], k[3:], 0.5, keep)
    eye = np.repeat(np.eye(4, 8)[:, None], 2, 1)
    p = attention(q[3:], k[3:], eye, 0.5, keep)[..., :4]     # (query, head, key)
    np.testing.assert_allclose(w, [p[:, :2].sum((0, 1)), p[:, 2:].sum((0, 1))], rtol=1e-12)


def test_eviction_by_hand():
    s = P.Sequence(8, 1, 1)
    s.append(np.arange(6.0).reshape(6, 1, 1), -np.arange(6.0).reshape(6, 1, 1))
    s.weights[0, :6] = [0, 3, 1, 3, 9, 2]
    s.evict(3, recent=1, first=1)            # 0 (first), 5 (recent), and 4 (weight 9)
    assert s.len == 3 and s.evicted == 3
    assert s.positions[0, :3].tolist() == [0, 4, 5] and s.weights[0, :3].tolist() == [0, 9, 2]
    assert s.rows[0, :3, 0, 0].tolist() == [0, 4, 5] and s.rows[1, :3, 0, 0].tolist() == [0, -4, -5]
    s.append(np.full((2, 1, 1), 7.0), np.full((2, 1, 1), 8.0))
    assert s.positions[0, :5].tolist() == [0, 4, 5, 6, 7] and s.weights[0, 3:5].tolist() == [0, 0]
    s.weights[0, :5] = [1, 1, 1, 1, np.nan]
    s.evict(3)                               # ties: the lower slots; NaN last
    assert s.positions[0, :3].tolist() == [0, 4, 5] and s.evicted == 5


def test_append_writes_the_account_of_its_tokens_only():
    s = P.Sequence(8, 1, 1)
    s.weights[:], s.positions[:], s.evicted = 5, 70, 10
    s.append(np.zeros((2, 1, 1)), np.zeros((2, 1, 1)), start=4)              # len is 0
    assert s.len == 6 and s.weights[0].tolist() == [5, 5, 5, 5, 0, 0, 5, 5]
    assert s.positions[0].tolist() == [70, 70, 70, 70, 14, 15, 70, 70]


@pytest.mark.parametrize("lens,H,Hk,frame", [((5, 0, 300, 129), 4, 2, 1), ((1000,), 8, 1, 64), ((64, 65), 2, 2, None), ((), 1, 1, 1), ((0,), 1, 1, 3),
                                             ((1374 * 3, 1374), 16, 16, 1374)])
def test_packed_plan_covers_every_row_once(lens, H, Hk, frame):
    plan = E.packed_plan(lens, H, Hk, 64, frame=frame)
    assert plan.cu.tolist() == np.cumsum((0,) + lens).tolist()
    tiles = plan.tiles.numpy()
    seen, cost = set(), []
    G = H // Hk
    for tok, n, row, zero in tiles:
        b = [i for i, m in enumerate(lens) if m and plan.cu[i] == tok][0]
        assert n == lens[b] and row % plan.rows == 0 and 0 <= row < n * G and zero == 0
        seen.add((b, row))
        last = (min(row + plan.rows, n * G) - 1) // G
        cost.append(-(-(n if frame is None else min(n, (last // frame + 1) * frame)) // 64))
    assert len(seen) == len(tiles) == sum(-(-n * G // plan.rows) for n in lens)
    assert cost == sorted(cost, reverse=True)


def test_packed_refusals():
    for args, kw, msg in ((((3, -1), 2, 1, 64), {}, "lens"), (((1 << 28, 1), 2, 2, 64), {}, "lens"), (((3,), 3, 2, 64), {}, "heads"),
                          (((3,), 2, 1, 96), {}, "heads"), (((3,), 2, 0, 64), {}, "heads"), (((3,), 2, 1, 64), dict(frame=0), "frame"), (((3,), 2, 1, 64), dict(frame=1 << 31), "frame"),
                          (((1 << 27,), 16, 1, 64), {}, "rows"), (((1 << 20,), 4096, 1, 64), {}, "rows")):
        with pytest.raises(RuntimeError, match=msg):
            E.packed_plan(*args, **kw)
    plan = E.packed_plan((4, 5), 4, 2, 64)
    q, k = torch.zeros(10, 4, 64).half(), torch.zeros(10, 2, 64).half()
    for args, kw, msg in (((q, k, k, None), {}, "packed_plan"), ((q, k, k, plan._replace(tiles=plan.tiles.long())), {}, "tiles must be"),
                          ((q, k, k, plan._replace(tiles=plan.tiles[:, :3])), {}, "tiles must be"),
                          ((q.float(), k, k, plan), {}, "data type"), ((q[:, :3], k, k, plan), {}, "q must be"),
                          ((q, k.bfloat16(), k, plan), {}, "k must be"), ((q, k, k[:9], plan), {}, "v must be"),
                          ((q[:8], k[:8], k[:8], plan), {}, "8 tokens"), ((q[None], k, k, plan), {}, "q must be"),
                          ((q, k, k, plan), dict(scale=-1.0), "scale"), ((q, k, k, plan), dict(out=q.float()), "out must be"),
                          ((q, k, k, plan), dict(out=q[:, :1].expand(10, 4, 64)), "out must be"),
                          ((q, k, k, plan), {}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            E.packed_attention(*args, **kw)


def test_packed_grids_that_a_launch_refuses():
    """Very many short sequences: a workgroup of 256 threads for each row tile and key head, under 2^32 threads in all."""
    with pytest.raises(RuntimeError, match="row tiles"):
        E.packed_plan((1,) * 300000, 64, 64, 64)
    assert E.packed_plan((1,) * 262143, 64, 64, 64).tiles.shape[0] == 262143
    lib, st, p = _lib.load(), (C.c_int64 * 2)(128, 64), 1 << 20
    for n, Hk in ((1 << 24, 1), (1 << 18, 64), ((1 << 63) - 1, 2)):
        assert lib.qv_packed_attention(p, p, p, p, 0, p, n, 256, 1, 50, 64, Hk, 64, st, st, st, st, 0.1, None) == -1
        assert "row tiles" in lib.qv_last_error().decode()


def test_paged_rows_whose_join_would_not_launch_are_not_cut():
    """The join has a thread for 4 dims of each row of a key head, under 2^32 in all: no parts from there on."""
    need = _lib.load().qv_paged_attention_workspace
    for rows, D in (((1 << 27) - 8, 128), ((1 << 28) - 16, 64)):
        assert need(0, 1, rows, 1, 1, D, 100000, 100000) > 0 and need(0, 1, rows // 2, 2, 1, D, 100000, 100000) > 0
        assert need(0, 1, rows, 2, 2, D, 100000, 100000) > 0
    for rows, D in ((1 << 27, 128), (1 << 28, 64)):
        assert need(0, 1, rows, 1, 1, D, 100000, 100000) == 0 and need(0, 1, rows // 2, 2, 1, D, 100000, 100000) == 0


def test_evict_refuses_an_account_off_16_bytes():
    """It is read four tokens at a time."""
    lib, p = _lib.load(), 1 << 20
    for w, pos in ((p + 4, p), (p, p + 8)):
        assert lib.qv_paged_evict(p, p, p, p, p, w, pos, 2, 2, 64, 16, 4, 9, 30, 3, 2, p, 1 << 20, None) == -1
        assert "aligned" in lib.qv_last_error().decode()


def test_paged_refusals():
    for args, kw, msg in (((2, 2, 32, 100), {}, "head_dim"), ((0, 2, 64, 100), {}, "batch"), ((2, 0, 64, 100), {}, "kv_heads"),
                          ((2, 2, 64, 0), {}, "capacity"), ((2, 2, 64, 100), dict(page=24), "page"), ((2, 2, 64, 100), dict(page=8), "page"),
                          ((2, 2, 64, 100), dict(pages=0), "pages"), ((2, 2, 64, 100), dict(dtype=torch.float32), "dtype"),
                          ((2, 2, 64, (1 << 29) + 1), {}, "capacity")):
        with pytest.raises(RuntimeError, match=msg):
            PagedKVCache(*args, **kw, device="cpu")
    c = PagedKVCache(2, 2, 64, 100, page=32, track=True, device="cpu")
    assert c.capacity == 128 and c.table.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7]] and c.k_pages.shape == (8, 2, 32, 64)
    assert (PagedKVCache(2, 2, 64, 100, pages=5, device="cpu").table == -1).all()
    q, k, lens = torch.zeros(2, 5, 4, 64).half(), torch.zeros(2, 9, 2, 64).half(), torch.zeros(2, dtype=torch.int32)
    plan = E.packed_plan((4, 5), 4, 2, 64)
    for args, kw, msg in (((k, k.bfloat16()), {}, "v must be"), ((k.bfloat16(), k.bfloat16()), {}, "k must be"), ((k[:1], k[:1]), {}, "k must be"),
                          ((k, k[:, :8]), {}, "v must be"), ((k[..., :32], k), {}, "k must be"), ((k[0], k[0]), {}, "k must be"),
                          ((k, k), dict(counts=lens.long()), "counts"), ((k, k), dict(start=lens[:1]), "start"),
                          ((torch.zeros(2, 129, 2, 64).half(),) * 2, {}, "do not fit"), ((k, k), dict(plan=plan), "k must be"),
                          ((k[0], k[0]), dict(plan=plan, counts=lens), "plan"), ((k[0, :8], k[0, :8]), dict(plan=plan), "8 tokens"),
                          ((k[0], k[0]), dict(plan=plan._replace(cu=plan.cu.long())), "cu must be"),
                          ((k[0], k[0]), dict(plan=plan._replace(cu=plan.cu[:2])), "cu must be"),
                          ((k[0], k[0]), dict(plan=E.packed_plan((4,), 4, 2, 64)), "2 sequences"), ((k, k), {}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            c.append(*args, **kw)
    for args, kw, msg in (((q[:1],), {}, "q must be"), ((q.bfloat16(),), {}, "q must be"), ((torch.zeros(2, 5, 4, 128).half(),), {}, "q must be"),
                          ((q[:, :, :3],), {}, "not a multiple"), ((q,), dict(counts=lens.long()), "counts"), ((q,), dict(scale=float("inf")), "scale"),
                          ((q,), dict(out=q[:, :2]), "out must be"), ((q,), dict(longest=-1), "longest"), ((q,), {}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            c.attention(*args, **kw)
    for args, kw, msg in (((3,), dict(recent=2, first=2), "within keep"), ((3,), dict(recent=-1), "within keep"), ((-1,), {}, "within keep"),
                          ((3,), {}, "GPU only")):
        with pytest.raises(RuntimeError, match=msg):
            c.evict(*args, **kw)
    bare = PagedKVCache(2, 2, 64, 100, device="cpu")
    with pytest.raises(RuntimeError, match="track"):
        bare.evict(3)
    with pytest.raises(RuntimeError, match="track"):
        bare.attention(q, collect=True)


def test_paged_tensors_are_replaced_by_like_ones_only():
    c = PagedKVCache(2, 2, 64, 100, page=32, track=True, device="cpu")
    for name, bad in (("table", lambda t: t.long()), ("table", lambda t: t[:, :2]), ("table", lambda t: t.t().contiguous().t()),
                      ("lens", lambda t: t[:1]), ("lens", lambda t: t.tolist()), ("k_pages", lambda t: t[:3]), ("v_pages", lambda t: t.bfloat16()),
                      ("weights", lambda t: t.double()), ("weights", lambda t: None), ("positions", lambda t: t[:, :, :64]),
                      ("evicted", lambda t: t.long()), ("lens", lambda t: t.to("meta")),
                      ("weights", lambda t: torch.zeros(t.numel() + 1)[1:].view(t.shape))):
        was = getattr(c, name)
        with pytest.raises(RuntimeError, match=f"{name} must be"):
            setattr(c, name, bad(was))
        assert getattr(c, name) is was
    new = torch.ones_like(c.table)
    c.table = new
    assert c.table is new


def test_account_of_a_cache_that_keeps_none():
    """Nothing would check a tensor that is put there, and the kernels would take its pointer."""
    c = PagedKVCache(2, 2, 64, 100, device="cpu")
    for name in ("weights", "positions", "evicted"):
        with pytest.raises(RuntimeError, match=f"{name} belongs to a cache with track=True"):
            setattr(c, name, torch.zeros(3))
        assert getattr(c, name) is None
        setattr(c, name, None)
    with pytest.raises(RuntimeError, match="track"):
        c.attention(torch.zeros(2, 1, 4, 64).half(), collect=True)


def test_paged_length_hint(monkeypatch):
    """How many keys the attention's plan is laid out for.  No kernel runs here."""
    from qvggt_amd import kv_cache as M
    calls = []
    monkeypatch.setattr(M, "_on_gpu", lambda *t, what: 0)
    monkeypatch.setattr(M, "_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(M, "_stream", lambda dev: 0)
    monkeypatch.setattr(M, "_capturing", lambda: False)
    monkeypatch.setattr(M._lib, "call", lambda name, *args: calls.append((name, args)))
    q, k = torch.zeros(2, 5, 4, 64).half(), torch.zeros(2, 9, 2, 64).half()
    c = PagedKVCache(2, 2, 64, 4000, device="cpu", track=True)

    def keys(**kw):
        c.attention(q, **kw)
        name, args = calls[-1]
        assert name == "qv_paged_attention" and args[-2] == M._paged_workspace_bytes(0, 2, 5, 4, 2, 64, args[18], c.capacity)
        return args[18]

    assert keys() == 0 and keys(longest=700) == 700 and keys(longest=1 << 40) == c.capacity
    c.append(k, k)
    c.append(k, k, start=c.lens)
    assert keys() == 18
    c.evict(10)
    assert keys() == 10
    c.append(k, k, start=torch.zeros(2, dtype=torch.int32))
    assert keys() == c.capacity
    c.reset()
    assert keys() == 0
    c.append(k, k)
    monkeypatch.setattr(M, "_capturing", lambda: True)       # a graph's replays are not counted
    assert keys() == c.capacity and keys(longest=30) == 30
    c.append(k, k)
    monkeypatch.setattr(M, "_capturing", lambda: False)
    assert keys() == c.capacity


def test_paged_length_hint_and_graphs(monkeypatch):
    """What is captured has not run yet, and a graph that appends may do so any time: the host then knows no length."""
    from qvggt_amd import kv_cache as M
    calls, capturing = [], [False]
    monkeypatch.setattr(M, "_on_gpu", lambda *t, what: 0)
    monkeypatch.setattr(M, "_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(M, "_stream", lambda dev: 0)
    monkeypatch.setattr(M, "_capturing", lambda: capturing[0])
    monkeypatch.setattr(M._lib, "call", lambda name, *args: calls.append(args))
    q, k = torch.zeros(2, 5, 4, 64).half(), torch.zeros(2, 200, 2, 64).half()
    c = PagedKVCache(2, 2, 64, 4000, device="meta", track=True)    # as on a GPU

    def keys():
        c.attention(q)
        return calls[-1][18]

    c.append(k, k)
    capturing[0] = True                      # captured, not run: the tokens are all there
    c.evict(30)
    c.reset()
    capturing[0] = False
    assert keys() == 200
    c.evict(100)
    assert keys() == 100
    capturing[0] = True
    c.append(k, k)
    c.evict(30)
    capturing[0] = False
    assert keys() == c.capacity
    c.evict(30)                              # the graph may be replayed behind these
    assert keys() == c.capacity
    c.reset()
    assert keys() == c.capacity
    c.append(k, k)
    assert keys() == c.capacity


def test_reset_of_a_cache_on_the_host():
    c = PagedKVCache(2, 2, 64, 100, device="cpu", track=True)
    c.lens.fill_(3), c.evicted.fill_(4)
    c.reset()
    assert not c.lens.any() and not c.evicted.any()


def test_c_entries_refuse():
    """Bad arguments end at the C entries with a message, before any device work (pointers here are never followed)."""
    lib = _lib.load()
    st, odd = (C.c_int64 * 3)(64 * 8, 64, 64), (C.c_int64 * 3)(64 * 8, 60, 64)
    two, odd2, far = (C.c_int64 * 2)(128, 64), (C.c_int64 * 2)(128, 60), (C.c_int64 * 2)(1 << 25, 64)
    p = 1 << 20

    def refused(rc, what):
        assert rc == -1 and what in lib.qv_last_error().decode(), (rc, lib.qv_last_error())

    pack = lambda **kw: lib.qv_packed_attention(*{**dict(q=p, k=p, v=p, out=p, dt=0, tiles=p, n=3, rows=128, frame=1, T=50, H=4, Hk=2, D=64, qs=two, ks=two,
                                                         vs=two, os=two, scale=0.1, s=None), **kw}.values())
    for kw, what in ((dict(dt=2), "dtype"), (dict(D=96), "head_dim"), (dict(Hk=3), "shape"), (dict(scale=0.0), "scale"), (dict(frame=0), "frame"),
                     (dict(n=-1), "row tiles"), (dict(rows=64), "256 of 64 dims"), (dict(rows=256, D=128), "256 of 64 dims"), (dict(n=1 << 30), "row tiles"), (dict(q=p + 8), "aligned"), (dict(k=p + 8), "aligned"),
                     (dict(tiles=p + 8), "aligned"), (dict(qs=odd2), "strides"), (dict(ks=odd2), "strides"), (dict(vs=far), "token strides"),
                     (dict(v=None), "null"), (dict(tiles=None), "null"), (dict(out=None), "null"), (dict(qs=None), "null"), (dict(ks=None), "null"),
                     (dict(T=1 << 27, H=256, Hk=2), "rows")):
        refused(pack(**kw), what)
    assert pack(T=0) == 0 and pack(n=0) == 0
    app = lambda **kw: lib.qv_paged_append(*{**dict(k=p, v=p, kp=p, vp=p, table=p, start=p, lens=p, tick=p, counts=None, cu=None, ev=None, w=None,
                                                    pos=None, B=2, n=5, T=0, Hk=2, D=64, page=16, slots=4, pages=9, ks=st, vs=st, s=None),
                                             **kw}.values())
    for kw, what in ((dict(D=32), "head_dim"), (dict(page=24), "page"), (dict(page=8), "page"), (dict(slots=1 << 26), "cache shape"),
                     (dict(B=40000), "cache shape"), (dict(pages=1 << 31), "cache shape"), (dict(n=-1), "number of tokens"), (dict(T=-1), "number of tokens"),
                     (dict(lens=None), "null"), (dict(table=None), "null"), (dict(kp=None), "null"), (dict(k=None), "null"), (dict(ks=None), "null"),
                     (dict(counts=p, cu=p), "two ways"), (dict(w=p), "together"), (dict(ev=p, pos=p), "together"), (dict(ks=odd), "strides"),
                     (dict(k=p + 2), "aligned"), (dict(vp=p + 8), "aligned")):
        refused(app(**kw), what)
    assert app(B=0) == 0
    att = lambda **kw: lib.qv_paged_attention(*{**dict(q=p, out=p, dt=0, kp=p, vp=p, table=p, lens=p, counts=None, causal=0, w=None, B=1, Lq=5, H=4,
                                                       Hk=2, D=64, page=16, slots=4, pages=9, keys=50, qs=st, os=st, scale=0.1, ws=None, wb=0, s=None),
                                                **kw}.values())
    for kw, what in ((dict(dt=2), "dtype"), (dict(D=32), "head_dim"), (dict(page=48), "page"), (dict(slots=1 << 26), "cache"), (dict(lens=None), "null"),
                     (dict(table=None), "null"), (dict(kp=None), "null"), (dict(kp=p + 8), "aligned"), (dict(qs=odd), "strides"), (dict(H=5), "shape"),
                     (dict(scale=-1.0), "scale"), (dict(w=p), "workspace"), (dict(w=p, ws=p, wb=79), "workspace"), (dict(B=70000), "grid")):
        refused(att(**kw), what)
    assert att(B=0) == 0 and att(Lq=0) == 0
    need = lib.qv_paged_attention_workspace
    assert need(0, 1, 1, 8, 1, 96, 5000, 5008) == 0 and need(1, 1, 1, 8, 3, 64, 5000, 5008) == 0
    assert need(0, 1, 1, 8, 1, 64, 64, 64) == 0 and need(0, 1, 1, 8, 1, 64, 64, -1) == 0
    assert need(0, 1, 1, 8, 1, 64, 100000, 100000) > 0
    # with what is received: the scores of all slots, up to 1 GiB of them, else log2 of the rows' sums
    assert need(1, 1, 1, 8, 1, 64, 64, 64) >= 8 * 64 * 4 and need(1, 1, 1, 8, 1, 64, 64, 1 << 25) >= 1 << 30
    assert 0 < need(1, 1, 1, 8, 1, 64, 64, (1 << 25) + 16) < 1 << 20
    ev = lambda **kw: lib.qv_paged_evict(*{**dict(kp=p, vp=p, table=p, lens=p, ev=p, w=p, pos=p, B=2, Hk=2, D=64, page=16, slots=4, pages=9, keep=30,
                                                  recent=3, first=2, ws=p, wb=1 << 20, s=None), **kw}.values())
    for kw, what in ((dict(D=32), "head_dim"), (dict(page=20), "page"), (dict(keep=4), "within keep"), (dict(keep=-1, recent=0, first=0), "within keep"),
                     (dict(recent=-1), "within keep"), (dict(first=(1 << 63) - 1), "within keep"), (dict(lens=None), "null"), (dict(w=None), "null"),
                     (dict(ws=None), "workspace"), (dict(wb=100), "workspace"), (dict(vp=p + 8), "aligned")):
        refused(ev(**kw), what)
    assert ev(B=0) == 0 and ev(keep=64) == 0
    need = lib.qv_paged_evict_workspace
    assert need(2, 2, 64, 64) == 0 and need(2, 2, 64, -1) == 0 and need(2, 3, 64, 60) == 256 + 6 * 4 * 8
