"""cross_attention and Int8KVCache.attention against the float64 oracle.

Bound for one output, with w_j the exact weights, u_p and u the half steps of
the probabilities (fp16 2^-11; bf16 2^-8) and of the output: the same rounded
probabilities form numerator and sum, so an error d_j of p_j moves the quotient by
w_j d_j (v_j - out): at most (u_p + 2 e) sum_j w_j |v_j - out|, itself at most
(u_p + 2 e) sqrt(sum_j w_j v_j^2 - out^2) as the weights sum to one, where e bounds the
absolute error of a score: fp32 sums of D products, (D + 4) 2^-24 sum |q k| scale, and
three fp32 roundings of its size.  fp16 probabilities below 2^-14 are off by 2^-25
each, where the largest of a row is 2^7 at least: 2^-32 of the sum.  Sums of N terms add N 2^-24 of their size.  Last,
the output's rounding.
"""
import math

import numpy as np
import pytest
import torch

from oracle import streaming as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def _close(got, q, k, v, scale=None, keep=None, p_type=None, rows=None):
    """One sequence: got, q (Lq, H, D), k, v (Lk, Hk, D)."""
    p_type = p_type or q.dtype
    u, up = HALF_STEP[got.dtype], HALF_STEP[p_type]
    got, q, k, v = (t.double().cpu().numpy() for t in (got, q, k, v))
    if rows is not None:
        got, q = got[rows], q[rows]
        keep = keep if keep is None or keep.ndim == 1 else keep[rows]
    D, G = q.shape[2], q.shape[1] // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    ref = O.attention(q, k, v, scale, keep)
    assert got.shape == ref.shape
    keep = np.broadcast_to(np.ones(len(k), bool) if keep is None else keep, (len(q), len(k)))
    n = len(k)
    for h in range(q.shape[1]):
        some = keep.any(0)
        kk, vv, kp = k[some][:, h // G], v[some][:, h // G], keep[:, some]
        if not some.any():
            assert not got[:, h].any()
            continue
        s = np.where(kp, q[:, h] @ kk.T * scale, -np.inf)
        w = np.exp(s - np.maximum(s.max(1, keepdims=True), -1e300))
        w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
        spread = np.sqrt(np.maximum(w @ vv ** 2 - ref[:, h] ** 2, 0)) + 1e-7 * np.abs(vv).max()
        size = np.where(kp, np.abs(q[:, h]) @ np.abs(kk).T, 0).max(1, keepdims=True) * scale
        e = ((D + 4) * 2.0 ** -24 + 3 * 2.0 ** -24) * size + 2.0 ** -21
        dev = np.abs(vv).max() * 2
        tol = ((up + 2 * e) * spread * 1.01 + (n * 2.0 ** -32 * dev if p_type == F16 else 0)
               + (n + 16) * 2.0 ** -24 * (w @ np.abs(vv)) + u * np.abs(ref[:, h]) * 1.01 + 2.0 ** -25)
        err = np.abs(got[:, h] - ref[:, h])
        assert (err <= tol).all(), (h, np.nanmax(err), np.nanmax(err / tol))


def _rand(gpu, seed, *shape, dtype=F16, sharp=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=gpu) * sharp).to(dtype)


def _qkv(gpu, seed, B, Lq, Lk, H, Hk, D, dtype, sharp=1.0):
    return (_rand(gpu, seed, B, Lq, H, D, dtype=dtype, sharp=sharp), _rand(gpu, seed + 1, B, Lk, Hk, D, dtype=dtype),
            _rand(gpu, seed + 2, B, Lk, Hk, D, dtype=dtype))


# ------------------------------------------------------------------- cross
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lq,Lk,H,Hk", [
    (1, 1, 1, 1), (1, 64, 2, 1), (1, 65, 4, 4), (1, 700, 8, 2), (5, 33, 6, 1), (7, 31, 4, 1), (8, 129, 4, 1), (32, 63, 1, 1),
    (33, 64, 1, 1), (11, 200, 3, 1), (64, 1, 2, 2), (100, 127, 2, 1), (128, 128, 1, 1), (129, 320, 2, 2), (300, 500, 2, 1),
    (513, 190, 1, 1)])
def test_cross(gpu, Lq, Lk, H, Hk, D, dtype):
    """One query to several row tiles of each form, key lengths around the tiles, shared heads."""
    from qvggt_amd import awq_inference_engine as E
    q, k, v = _qkv(gpu, Lq + Lk, 2, Lq, Lk, H, Hk, D, dtype)
    out = E.cross_attention(q, k, v)
    assert out.shape == q.shape and torch.isfinite(out).all()
    for b in range(2):
        _close(out[b], q[b], k[b], v[b])


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("Lq,H", [(1, 4), (50, 4), (300, 2)])
@pytest.mark.parametrize("sharp", [5.0, 40.0])
def test_cross_sharp_scores(gpu, Lq, H, D, dtype, sharp):
    """Scores up to hundreds: the running maximum moves between tiles, splits and waves."""
    from qvggt_amd import awq_inference_engine as E
    q, k, v = _qkv(gpu, 3, 1, Lq, 1500, H, 2, D, dtype, sharp)
    _close(E.cross_attention(q, k, v)[0], q[0], k[0], v[0])
    up = torch.linspace(0, 3, 1500, device=gpu).view(1, -1, 1, 1)      # the largest key last
    k = (k.abs() * up).to(dtype)
    _close(E.cross_attention(q.abs(), k, v, scale=0.05)[0], q[0].abs(), k[0], v[0], scale=0.05)


@pytest.mark.parametrize("Lq,H,Hk", [(1, 2, 1), (40, 2, 2), (150, 2, 1)])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, F16), (64, BF16)])
def test_cross_masks_and_lengths(gpu, Lq, H, Hk, D, dtype):
    """Left-out keys hold NaN and infinities; empty sequences; masks that leave one key, a tile, nothing."""
    from qvggt_amd import awq_inference_engine as E
    B, Lk = 7, 300
    q, k, v = _qkv(gpu, 17, B, Lq, Lk, H, Hk, D, dtype)
    lens = torch.tensor([300, 0, 1, 64, 65, 299, 300], dtype=torch.int32, device=gpu)
    keep = torch.rand(B, Lk, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)) > 0.3
    keep[0, 64:192] = False
    keep[3] = False
    keep[5] = False
    keep[5, 150] = True
    keep[6] = True
    inside = torch.arange(Lk, device=gpu) < lens[:, None]
    for use_lens, use_mask in ((True, False), (False, True), (True, True)):
        seen = (inside if use_lens else torch.ones_like(keep)) & (keep if use_mask else torch.ones_like(keep))
        kk, vv = k.clone(), v.clone()
        kk[~seen], vv[~seen] = float("nan"), float("inf")
        vv[~seen] = torch.where(torch.rand(vv[~seen].shape, device=gpu) > 0.5, float("nan"), float("-inf")).to(dtype)
        out = E.cross_attention(q, kk, vv, kv_lens=lens if use_lens else None, key_mask=keep if use_mask else None)
        for b in range(B):
            _close(out[b], q[b], k[b], v[b], keep=seen[b].cpu().numpy())
    out = E.cross_attention(q, k, v, kv_lens=lens * 1000 - 5)           # drawn into 0 .. Lk
    assert torch.equal(out, E.cross_attention(q, k, v, kv_lens=(lens > 0).int() * Lk))
    wide = torch.zeros(B, 2 * Lk, dtype=torch.bool, device=gpu)
    wide[:, ::2] = keep
    assert torch.equal(E.cross_attention(q, k, v, key_mask=wide[:, ::2]), E.cross_attention(q, k, v, key_mask=keep))
    assert not E.cross_attention(q, k[:, :0], v[:, :0]).any()
    assert E.cross_attention(q[:0], k[:0], v[:0]).shape == (0, Lq, H, D)
    assert E.cross_attention(q[:, :0], k, v).shape == (B, 0, H, D)


@pytest.mark.parametrize("Lq,Lk,H,Hk,D,dtype", [(1, 20000, 2, 1, 64, F16), (1, 9000, 8, 1, 128, BF16), (20, 5000, 1, 1, 64, BF16),
                                               (60, 7000, 2, 1, 128, F16), (200, 4000, 2, 1, 64, F16)])
def test_cross_split_keys(gpu, Lq, Lk, H, Hk, D, dtype):
    """Few rows over many keys: the key range is split and joined; repeatable, and right when a split is empty or masked."""
    from qvggt_amd import _lib
    from qvggt_amd import awq_inference_engine as E
    assert _lib.load().qv_attention_kv_workspace(0, 1, Lq, H, Hk, D, Lk) > 0
    q, k, v = _qkv(gpu, 23, 1, Lq, Lk, H, Hk, D, dtype, 3.0)
    out = E.cross_attention(q, k, v)
    _close(out[0], q[0], k[0], v[0])
    assert torch.equal(out, E.cross_attention(q, k, v))
    for n in (1, 70, Lk // 2):
        lens = torch.tensor([n], dtype=torch.int32, device=gpu)
        _close(E.cross_attention(q, k, v, kv_lens=lens)[0], q[0], k[0, :n], v[0, :n])
    keep = torch.zeros(1, Lk, dtype=torch.bool, device=gpu)
    keep[0, Lk - 3] = True
    assert torch.equal(E.cross_attention(q, k, v, key_mask=keep)[0], v[0, Lk - 3].repeat_interleave(H // Hk, 0).expand(Lq, H, D))
    assert not E.cross_attention(q, k, v, key_mask=keep & False).any()


@pytest.mark.parametrize("B,H,Lk,D", [(8, 16, 9001, 64), (2, 64, 5003, 128)])
def test_cross_split_keys_of_many_heads(gpu, B, H, Lk, D):
    """One query of 128 heads over more keys than the caches hold: split in two, lengths of all kinds."""
    from qvggt_amd import awq_inference_engine as E
    assert E._kv_workspace_bytes(0, B, 1, H, H, D, Lk) > 0
    q, k, v = _qkv(gpu, 27, B, 1, Lk, H, H, D, F16, 3.0)
    out = E.cross_attention(q, k, v)
    for b in (0, B - 1):
        _close(out[b], q[b], k[b], v[b])
    lens = torch.tensor([(1, Lk // 2, Lk // 2 + 70, 0, Lk, 64, 65, 5000)[b] for b in range(B)], dtype=torch.int32, device=gpu)
    out = E.cross_attention(q, k, v, kv_lens=lens)
    for b, n in enumerate(lens.tolist()):
        _close(out[b], q[b], k[b, :n], v[b, :n])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Lq,Lk", [(1, 1, 1374), (3, 40, 300), (1, 300, 1374), (1, 1374, 1374)])
def test_cross_weights_sum_to_one(gpu, B, Lq, Lk, dtype):
    """One value vector for all keys comes back exactly: sums and products take the
    same rounded probabilities, 1374 terms at 2^-23 are under half a step (and a
    join of splits adds a few roundings of 2^-24)."""
    from qvggt_amd import awq_inference_engine as E
    q, k, v = _qkv(gpu, 29, B, Lq, Lk, 4, 4, 64, dtype, 4.0)
    v[:] = v[:, :1].clone()
    assert torch.equal(E.cross_attention(q, k, v), v[:, :1].expand(B, Lq, 4, 64))


@pytest.mark.parametrize("Lq,D", [(1, 64), (40, 128), (200, 64)])
def test_cross_strides(gpu, Lq, D):
    """Fused buffers, heads before tokens, expanded states, unaligned rows, an out of its own layout."""
    from qvggt_amd import awq_inference_engine as E
    B, Lk, H, Hk = 2, 150, 4, 2
    q, k, v = _qkv(gpu, 31, B, Lq, Lk, H, Hk, D, F16)
    want = E.cross_attention(q, k, v)
    fused = torch.cat([k, v], 2)
    perm = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    odd = lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2]
    gap = lambda t: torch.nn.functional.pad(t, (0, 8, 0, 1))[:, :, :-1, :-8]
    for qq, kk, vv in ((q, fused[:, :, :Hk], fused[:, :, Hk:]), (perm(q), perm(k), perm(v)), (odd(q), odd(k), v),
                       (gap(q), k, gap(v)), (q.transpose(2, 3).contiguous().transpose(2, 3), k, v)):
        assert torch.equal(E.cross_attention(qq, kk, vv), want)
    big = torch.full((B, H, Lq, D + 4), 7.0, dtype=F16, device=gpu)
    out = big.transpose(1, 2)[..., :D]
    assert E.cross_attention(q, k, v, out=out) is out and torch.equal(out, want) and (big[..., D:] == 7).all()
    one = E.cross_attention(q, k[:1].expand(B, Lk, Hk, D), v[:1].expand(B, Lk, Hk, D))
    assert torch.equal(one[0], want[0])
    _close(one[1], q[1], k[0], v[0])
    same = k[:, :1].expand(B, Lk, Hk, D)                                # one token repeated
    _close(E.cross_attention(q, same, v)[1], q[1], same[1], v[1])


@pytest.mark.parametrize("Lq", [1, 40, 200])
def test_smaller_workspaces(gpu, monkeypatch, Lq):
    """With less workspace than asked for the keys are split less, down to not at all."""
    from qvggt_amd import awq_inference_engine as E
    q, k, v = _qkv(gpu, 33, 2, Lq, 5000, 2, 1, 64, F16, 3.0)
    full = E._kv_workspace_bytes(0, 2, Lq, 2, 1, 64, 5000)
    want = E.cross_attention(q, k, v)
    one = 2 * Lq * 2 * (64 * 4 + 8)
    assert full % one == 0 and full > 3 * one
    for size in (3 * one + 5, one, 16, 0):
        monkeypatch.setattr(E, "_kv_workspace_bytes", lambda *shape: size)
        out = E.cross_attention(q, k, v)
        for b in range(2):
            _close(out[b], q[b], k[b], v[b])
    monkeypatch.undo()
    assert torch.equal(E.cross_attention(q, k, v), want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Lq", [1, 9, 64, 300])
def test_cross_and_cached_agree(gpu, Lq, dtype):
    """The cache's values as 16-bit keys and values give what the cache gives: both against
    the oracle, causal rows as a mask."""
    from qvggt_amd import awq_inference_engine as E
    c = _cache(gpu, 51, 1, (700,), 2, 64, F16)
    k, v = c.values(700, dtype=F16)
    q = _rand(gpu, 52, 1, Lq, 4, 64)
    _close(E.cross_attention(q, k, v)[0], q[0], k[0], v[0])
    _check_cached(c.attention(q.to(dtype)), q.to(dtype), c)


def test_cross_long_offsets(gpu):
    """Keys and values whose offsets pass 32 bits (a 5.2 GB buffer, 65536 elements from token to token)."""
    from qvggt_amd import awq_inference_engine as E
    Lk, ts = 40000, 65536
    buf = torch.empty(Lk * ts, dtype=F16, device=gpu)
    rows = buf.view(1, Lk, ts // 64, 64)
    g = torch.Generator(device=gpu).manual_seed(1)
    kv = torch.randn(2, Lk, 64, generator=g, device=gpu).half()
    k, v = rows[:, :, 3:4], rows[:, :, 900:901]
    k.copy_(kv[0].view(1, Lk, 1, 64))
    v.copy_(kv[1].view(1, Lk, 1, 64))
    for Lq in (1, 40):
        q = _rand(gpu, Lq, 1, Lq, 1, 64, sharp=4.0)
        out = E.cross_attention(q, k, v)
        assert torch.equal(out, E.cross_attention(q, kv[0].view(1, Lk, 1, 64), kv[1].view(1, Lk, 1, 64)))
        _close(out[0], q[0], k[0], v[0])


def test_cross_non_finite_inputs_reach_their_outputs(gpu):
    from qvggt_amd import awq_inference_engine as E
    for Lq in (2, 100):
        q, k, v = _qkv(gpu, 37, 2, Lq, 200, 2, 2, 64, F16)
        q[0, 1, 0, 5] = float("nan")
        v[1, 150, 1, 9] = float("nan")
        bad = ~torch.isfinite(E.cross_attention(q, k, v))
        want = torch.zeros_like(bad)
        want[0, 1, 0] = True
        want[1, :, 1, 9] = True
        assert torch.equal(bad, want)


def test_cross_stream_and_graph(gpu):
    """Two graphs and eager calls share nothing: replayed in turn, each gives the eager result of its inputs."""
    from qvggt_amd import awq_inference_engine as E
    a, b = _qkv(gpu, 41, 1, 1, 6000, 4, 2, 64, F16), _qkv(gpu, 43, 1, 70, 3000, 4, 2, 64, F16)
    graphs, outs = [], []
    for args in (a, b):
        E.cross_attention(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(E.cross_attention(*args))
        graphs.append(graph)
    for i in range(4):
        for t in (*a, *b):
            t.mul_(0.9)
        want = [E.cross_attention(*args) for args in (a, b)]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = E.cross_attention(*a)
    want = E.cross_attention(*a)
    torch.cuda.synchronize()
    assert torch.equal(other, want)


# ------------------------------------------------------------------- cached
def _cache(gpu, seed, B, lens, Hk, D, dtype, size=1.0, capacity=None):
    from qvggt_amd.kv_cache import Int8KVCache
    n = max(lens)
    c = Int8KVCache(B, Hk, D, capacity or n, device=gpu)
    k, v = _rand(gpu, seed, B, n, Hk, D, dtype=dtype), _rand(gpu, seed + 1, B, n, Hk, D, dtype=dtype, sharp=size)
    c.append(k, v, counts=torch.tensor(lens, dtype=torch.int32, device=gpu))
    return c


def _check_cached(out, q, cache, causal=False, counts=None, scale=None, rows=None):
    k, v = cache.values(int(cache.lens.max()))
    for b, n in enumerate(cache.lens.tolist()):
        nq = q.shape[1] if counts is None else counts[b]
        keep = None
        if causal:
            keep = np.arange(n) <= (n - nq + np.arange(nq))[:, None]
        if nq:
            _close(out[b, :nq], q[b, :nq], k[b, :n], v[b, :n], scale=scale, keep=keep, p_type=F16, rows=rows)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Lq,lens,H,Hk", [
    (1, (1, 64), 1, 1), (1, (65, 700), 8, 2), (1, (0, 200), 4, 4), (5, (5, 33), 6, 1), (8, (129, 20), 4, 1), (32, (63, 40), 1, 1),
    (33, (64, 33), 1, 1), (11, (200, 11), 3, 1), (64, (64, 100), 2, 2), (100, (127, 400), 2, 1), (129, (320, 129), 2, 2),
    (300, (500, 301), 2, 1), (40, (10, 70), 2, 1)])
def test_cached(gpu, Lq, lens, H, Hk, D, dtype, causal):
    """Both forms, lengths around the blocks, fewer tokens than queries (causal rows that see nothing), shared heads."""
    c = _cache(gpu, Lq + H, 2, lens, Hk, D, dtype, capacity=max(lens) + 100)
    q = _rand(gpu, 5, 2, Lq, H, D, dtype=dtype, sharp=2.0)
    out = c.attention(q, causal=causal)
    assert out.dtype == dtype and torch.isfinite(out).all()
    _check_cached(out, q, c, causal)


@pytest.mark.parametrize("Lq,n,H,Hk,D,dtype,causal", [
    (1, 20000, 2, 1, 64, F16, True), (1, 9000, 8, 1, 128, BF16, False), (20, 5000, 1, 1, 64, BF16, True),
    (60, 7000, 2, 1, 128, F16, True), (200, 4000, 2, 1, 64, F16, False), (300, 3000, 2, 1, 128, BF16, True)])
def test_cached_split_keys(gpu, Lq, n, H, Hk, D, dtype, causal):
    from qvggt_amd import _lib
    assert _lib.load().qv_attention_kv_workspace(1, 2, Lq, H, Hk, D, n) > 0
    c = _cache(gpu, 7, 2, (n, 333), Hk, D, dtype)
    q = _rand(gpu, 8, 2, Lq, H, D, dtype=dtype, sharp=4.0)
    out = c.attention(q, causal=causal)
    rows = np.unique(np.linspace(0, Lq - 1, 40).astype(int))
    _check_cached(out, q, c, causal, rows=rows)
    assert torch.equal(out, c.attention(q, causal=causal))
    c._bound = 0                                          # the hint only: one range a row tile
    _check_cached(c.attention(q, causal=causal), q, c, causal, rows=rows)


@pytest.mark.parametrize("Lq,H", [(3, 4), (50, 2), (200, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_cached_counts_leave_the_rest(gpu, Lq, H, causal):
    """A padded batch: rows behind a sequence's queries stay as they were (zero in a new tensor)."""
    c = _cache(gpu, 9, 4, (300, 64, 5, 0), 2, 64, F16, capacity=400)
    q = _rand(gpu, 10, 4, Lq, H, 64)
    counts = [Lq, 1, 0, 2]
    q[1, 1:], q[2], q[3, 2:] = float("nan"), float("nan"), float("nan")
    ct = torch.tensor(counts, dtype=torch.int32, device=gpu)
    out = torch.full_like(q, 5.0)
    c.attention(q, causal=causal, counts=ct, out=out)
    _check_cached(out, q, c, causal, counts)
    new = c.attention(q, causal=causal, counts=ct)
    for b, n in enumerate(counts):
        assert (out[b, n:] == 5).all() and not new[b, n:].any() and torch.equal(new[b, :n], out[b, :n])
    assert torch.equal(c.attention(q, counts=ct * 100 - 1, causal=causal)[0], c.attention(q, causal=causal)[0])


@pytest.mark.parametrize("Lq", [1, 100])
@pytest.mark.parametrize("dtype,sizes", [(F16, (1.0, 1e-4, 1e4, 0.0, 3e-3, 1e4, 1e-6)), (BF16, (1e-30, 1.0, 1e30, 1e-30, 1e25, 1.0, 0.0)),
                                         (F16, (0.0,) * 7), (BF16, (1e30, 1e-35) * 3 + (1e-35,))])
@pytest.mark.parametrize("D", [64, 128])
def test_cached_value_scales_apart(gpu, Lq, dtype, sizes, D):
    """Blocks of values far apart in size, in any order, queries that look at one of them only: O's unit moves along.
    Relative to the largest value of the sequence, at most 2^-60 is lost (units stay within that range)."""
    from qvggt_amd.kv_cache import Int8KVCache
    n = 64 * len(sizes)
    c = Int8KVCache(1, 1, D, n, device=gpu)
    k, v = _rand(gpu, 1, 1, n, 1, D, dtype=dtype), _rand(gpu, 2, 1, n, 1, D, dtype=torch.float32)
    v = (v * torch.tensor(sizes, device=gpu).repeat_interleave(64).view(1, n, 1, 1)).to(dtype)
    c.append(k, v)
    q = _rand(gpu, 3, 1, Lq, 1, D, dtype=dtype)
    q[0, 0, 0] = k[0, 64 * 4 + 7, 0] * 8                   # this row sees block 4 almost alone
    out = c.attention(q)
    assert torch.isfinite(out).all()
    kk, vv = c.values()
    top = float(vv.abs().max())
    if top == 0:
        assert not out.any()
        return
    ref = O.attention(q[0].double().cpu().numpy(), kk[0].double().cpu().numpy(), vv[0].double().cpu().numpy(), D ** -0.5)
    w = O.attention(q[0].double().cpu().numpy(), kk[0].double().cpu().numpy(), vv[0].abs().double().cpu().numpy(), D ** -0.5)
    err = np.abs(out[0].double().cpu().numpy() - ref)
    # u_p and score errors against the sizes that the row weighs; fp16 tails 2^-32 of each value's size
    tol = (4 * 2.0 ** -11) * w + HALF_STEP[dtype] * np.abs(ref) * 1.01 + n * 2.0 ** -32 * top + 2.0 ** -25 * (dtype == F16)
    assert (err <= tol).all(), (err / tol).max()


def test_cached_keys_of_extreme_size(gpu):
    """Scores from huge keys and tiny queries (and the reverse) that meet at ordinary size."""
    from qvggt_amd.kv_cache import Int8KVCache
    for size in (1e30, 1e-30):
        for Lq in (1, 70):
            c = Int8KVCache(1, 1, 64, 200, device=gpu)
            k, v = _rand(gpu, 1, 1, 200, 1, 64, dtype=BF16, sharp=size), _rand(gpu, 2, 1, 200, 1, 64, dtype=BF16)
            c.append(k, v)
            q = _rand(gpu, 3, 1, Lq, 1, 64, dtype=BF16, sharp=1 / size)
            _check_cached(c.attention(q), q, c)


def test_cached_marked_block(gpu):
    """A NaN that was appended comes back in its head, in whatever sees its block."""
    for Lq, H in ((1, 4), (80, 2)):
        for which in (0, 1):
            c = _cache(gpu, 12, 2, (200, 200), 2, 64, F16, capacity=300)
            kv = [_rand(gpu, 13 + i, 2, 1, 2, 64) for i in range(2)]
            kv[which][1, 0, 1, 3] = float("nan")
            c.append(*kv)
            q = _rand(gpu, 15, 2, Lq, H, 64)
            bad = ~torch.isfinite(c.attention(q))
            want = torch.zeros_like(bad)
            want[1, :, H // 2:] = True
            assert torch.equal(bad, want)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lq,past", [(1, 191), (3, 190), (80, 190), (300, 190), (80, 4000), (300, 9000)])
def test_cached_marked_block_behind_causal_queries(gpu, Lq, past, D, which):
    """A NaN of the last token marks its block: queries that see a token of the block come
    back NaN, the ones before it as if it were not there, tiles they share included."""
    c = _cache(gpu, 61, 1, (past,), 2, D, F16, capacity=past + Lq)
    kv = [_rand(gpu, 62 + i, 1, Lq, 2, D) for i in range(2)]
    kv[which][0, -1, 1, 3] = float("nan")
    c.append(*kv)
    q = _rand(gpu, 64, 1, Lq, 4, D)
    out = c.attention(q, causal=True)
    last = past + Lq - 1
    sees = past + torch.arange(Lq, device=gpu) >= last // 64 * 64
    want = torch.zeros(1, Lq, 4, D, dtype=torch.bool, device=gpu)
    want[:, sees, 2:] = True
    assert torch.equal(torch.isnan(out), want) and torch.isfinite(out[~want]).all()
    clean = (~sees).nonzero()[:, 0].cpu().numpy()
    if len(clean):
        _check_cached(out, q, c, causal=True, rows=clean)


def test_cached_scale_argument_and_strides(gpu):
    c = _cache(gpu, 21, 2, (150, 90), 2, 128, F16)
    for Lq in (1, 60):
        q = _rand(gpu, 22, 2, Lq, 6, 128)
        want = c.attention(q, scale=0.3)
        _check_cached(want, q, c, scale=0.3)
        big = torch.nn.functional.pad(q, (0, 8, 1, 2))[:, :, 1:-2, :-8]
        assert torch.equal(c.attention(big, scale=0.3), want)
        out = torch.empty(2, 6, Lq, 128, dtype=F16, device=gpu).transpose(1, 2)
        assert c.attention(q, scale=0.3, out=out) is out and torch.equal(out, want)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, F16), (64, BF16)])
@pytest.mark.parametrize("Lq", [1, 50, 200])
def test_cached_scale_of_zero(gpu, Lq, D, dtype):
    """A block whose scale is 0 holds zeros, whatever its codes are (loaded ones may be anything): keys, values, both."""
    c = _cache(gpu, 71, 1, (500,), 2, D, dtype)
    kc, ks, vc, vs, lens = c.save_codes()
    ks[0, 1], ks[0, 3, 0], ks[0, 7, 1] = 0, 0, 0
    vs[0, 2], vs[0, 3, 0], vs[0, 7, 0] = 0, 0, 0
    c.load_codes(kc, ks, vc, vs, lens)
    assert c.k_codes[0, :, 1].any() and not c.values()[0][0, 64:128].any()
    q = _rand(gpu, 72, 1, Lq, 4, D, dtype=dtype, sharp=3.0)
    for causal in (False, True):
        _check_cached(c.attention(q, causal=causal), q, c, causal)


def _check_blocks_apart(out, q, c, causal, lost=0.0):
    """Every key of a block has the same score, so its rounded probabilities are equal and cancel; blocks that a row
    does not look at weigh under 2^-100.  What is left are fp32 sums and the output's rounding, and what the sizes
    in a row's sight may lose where they pass 2^60: lost times the largest value that it sees."""
    k, v = (t[0].double().cpu().numpy() for t in c.values(int(c.lens[0])))
    n, Lq = len(k), q.shape[1]
    keep = np.arange(n) <= (n - Lq + np.arange(Lq))[:, None] if causal else None
    q, got, u = q[0].double().cpu().numpy(), out[0].double().cpu().numpy(), HALF_STEP[out.dtype]
    assert np.isfinite(got).all()
    ref, size = (O.attention(q, k, x, q.shape[2] ** -0.5, keep) for x in (v, np.abs(v)))
    tol = (n + 16) * 2.0 ** -24 * size + u * np.abs(ref) * 1.01 + (2.0 ** -25 if out.dtype == F16 else 0)
    if lost:
        tol += lost * np.where(keep, np.abs(v).max((1, 2)), 0).max(1)[:, None, None]
    err = np.abs(got - ref)
    assert (err <= tol).all(), (np.argwhere(err > tol)[:5], np.nanmax(err / np.maximum(tol, 1e-300)))


def _blocks_apart(gpu, sizes, Lq, H, D, dtype, looks=True):
    """A cache of one key head, block t's keys the unit vector t (times 30), its values of size sizes[t]; query i looks at
    block i % blocks (some rows at none)."""
    from qvggt_amd.kv_cache import Int8KVCache
    nb = len(sizes)
    n = 64 * nb - 5
    c = Int8KVCache(1, 1, D, n, device=gpu)
    k = torch.zeros(1, n, 1, D, device=gpu)
    k[0, torch.arange(n), 0, torch.arange(n) // 64] = 30.0
    v = _rand(gpu, 2, 1, n, 1, D, dtype=torch.float32) * torch.tensor(sizes, device=gpu).repeat_interleave(64)[:n].view(1, n, 1, 1)
    c.append(k.to(dtype), v.to(dtype))
    q = torch.zeros(1, Lq, H, D, device=gpu)
    if looks:
        i = torch.arange(Lq * H, device=gpu)
        q.view(Lq * H, D)[i, i % (nb + 1)] = 30.0          # dim nb: no block's
    return c, q.to(dtype)


@pytest.mark.parametrize("dtype,sizes", [
    (BF16, (1.0, 2.0 ** -50, 8.0, 2.0 ** -55, 2.0 ** -20, 2.0 ** -50, 2.0 ** -40)),
    (BF16, (2.0 ** -20, 2.0 ** 35, 2.0 ** -20, 2.0 ** 30, 2.0 ** -20, 1.0, 2.0 ** 35)),
    (BF16, (2.0 ** -105, 2.0 ** -60, 2.0 ** -100, 2.0 ** -90, 2.0 ** -60, 2.0 ** -110, 2.0 ** -70)),
    (F16, (2.0 ** -12, 2.0 ** 11, 2.0 ** -12, 1.0, 2.0 ** -12, 2.0 ** 11, 2.0 ** -3))])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Lq,H", [(9, 3), (50, 2), (300, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_cached_small_blocks_beside_large_ones(gpu, Lq, H, D, causal, dtype, sizes):
    """Rows that look at one block keep its values whatever the size of the others within 2^60, in any order."""
    c, q = _blocks_apart(gpu, sizes, Lq, H, D, dtype)
    _check_blocks_apart(c.attention(q, causal=causal), q, c, causal)


@pytest.mark.parametrize("sizes", [(1e-30, 1e30), (1e-33, 1e-11, 1e11, 1e33), (1e-33, 1e-33, 1e33, 1e33, 1e33), (1e20, 1e-10, 1e33)])
@pytest.mark.parametrize("Lq,H", [(9, 3), (50, 2), (60, 4), (110, 1), (110, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_cached_unseen_blocks_take_nothing(gpu, Lq, H, D, sizes):
    """Causal rows that share their tiles with a much larger later block, which they do not see: nothing of theirs is lost."""
    c, q = _blocks_apart(gpu, sizes, Lq, H, D, BF16, looks=False)
    _check_blocks_apart(c.attention(q, causal=True), q, c, True, lost=2.0 ** -60)


@pytest.mark.parametrize("Lq,H", [(1, 2), (50, 1), (200, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("split", [False, True])
def test_cached_tiny_values_of_many_tokens(gpu, Lq, H, D, split):
    """The smallest scale beside a sum of 8000 weights of 2^14.5: their quotient is no normal number, the result is.
    One value for all tokens comes back exactly (8000 terms at 2^-23 are under half a step)."""
    from qvggt_amd.kv_cache import Int8KVCache
    n = 8000
    c = Int8KVCache(1, 1, D, n, device=gpu)
    k, v = torch.zeros(1, n, 1, D, device=gpu), torch.full((1, n, 1, D), 2.0 ** -114, device=gpu)
    k[0, 64:, 0, 0] = 1.0
    c.append(k.bfloat16(), v.bfloat16())
    assert (c.v_scales[0, 0, :-(-n // 64)] == 2.0 ** -120).all()
    q = torch.zeros(1, Lq, H, D, device=gpu)
    q[..., 0] = 7.5 * math.log(2.0) * D ** 0.5
    if not split:
        c._bound = 0                                      # the hint only
    assert (c.attention(q.bfloat16()) == 2.0 ** -114).all()


def test_cached_long_offsets(gpu):
    """A cache whose heads lie past 4 GB: keys of zero everywhere but in the last tokens."""
    from qvggt_amd.kv_cache import Int8KVCache
    D, Hk, n = 128, 16, 2_300_000
    c = Int8KVCache(1, Hk, D, n, device=gpu)
    assert c.k_codes.numel() > 1 << 32
    k, v = _rand(gpu, 1, 1, 100, Hk, D), _rand(gpu, 2, 1, 100, Hk, D)
    at = torch.tensor([n - 100], dtype=torch.int32, device=gpu)
    c.append(k, v, start=at)
    kk, vv = c.values(100, first=at)
    for Lq in (1, 40):
        q = (k[:, :Lq] * 3).contiguous()                   # looks at one of the last tokens
        out = c.attention(q)[0].double().cpu()
        q64, k64, v64 = q[0].double().cpu(), kk[0].double().cpu(), vv[0].double().cpu()
        s = torch.einsum("qhd,khd->hqk", q64, k64) * D ** -0.5
        p = torch.exp(s)
        ref = torch.einsum("hqk,khd->qhd", p / (p.sum(-1, keepdim=True) + (n - 100)), v64)
        # a weight is off by 2^-11, the lost parts of the even keys by 2^-32 of the sum each
        size = torch.einsum("hqk,khd->qhd", p / (p.sum(-1, keepdim=True) + (n - 100)), v64.abs())
        tol = 4 * 2.0 ** -11 * size + 2.0 ** -11 * ref.abs() + n * 2.0 ** -32 * 2 * v64.abs().max() + 2.0 ** -25
        assert bool(((out - ref).abs() <= tol).all()), float(((out - ref).abs() / tol).max())
    del c


def test_stream_of_frames(gpu):
    """The operators together: frames of 1374 tokens rotated by (time, y, x), appended, attended to, against the
    same steps in 64 bits; then single tokens; one graph of a step, replayed."""
    from qvggt_amd import awq_inference_engine as E
    from qvggt_amd.aggregator import vggt_positions
    from qvggt_amd.kv_cache import Int8KVCache
    H, D, T, frames = 4, 64, 1374, 3
    plan = E.rope_axes_plan(D, (16, 24, 24), device=gpu)
    pairs = O.rope_pairs((16, 24, 24), "block")
    cache = Int8KVCache(1, H, D, (frames + 1) * T, device=gpu)
    ref = [O.Cache(cache.capacity, H, D) for _ in range(2)]
    yx = vggt_positions(1, gpu)

    def step(qkv, pos):
        qk = E.rope_axes(qkv[:, :2 * H], pos, plan)
        cache.append(qk[:, H:].unsqueeze(0), qkv[:, 2 * H:].unsqueeze(0))
        return qk, cache.attention(qk[:, :H].unsqueeze(0))[0]

    def check(qkv, pos, qk, out):
        want = O.rope_axes(qkv[:, :2 * H].double().cpu().numpy(), pos.cpu().numpy(), pairs)
        np.testing.assert_allclose(qk.double().cpu().numpy(), want, atol=2e-3, rtol=2.0 ** -10)
        ref[0].append(qk[:, H:].double().cpu().numpy())
        ref[1].append(qkv[:, 2 * H:].double().cpu().numpy())
        k, v = cache.values(ref[0].len)
        np.testing.assert_array_equal(k[0].cpu().numpy(), ref[0].values())
        np.testing.assert_array_equal(v[0].cpu().numpy(), ref[1].values())
        rows = np.unique(np.linspace(0, len(out) - 1, 24).astype(int))
        _close(out, qk[:, :H], k[0], v[0], p_type=F16, rows=rows)

    for f in range(frames):
        qkv = _rand(gpu, f, T, 3 * H, D)
        pos = torch.cat([torch.full((T, 1), f, dtype=torch.int32, device=gpu), yx], 1)
        check(qkv, pos, *step(qkv, pos))
    qkv = _rand(gpu, 99, 1, 3 * H, D)
    pos = torch.tensor([[frames, 0, 0]], dtype=torch.int32, device=gpu)
    check(qkv, pos, *step(qkv, pos))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qk, out = step(qkv, pos)
    for i in range(4):
        qkv.copy_(_rand(gpu, 100 + i, 1, 3 * H, D))
        pos[0, 1:] += 1
        graph.replay()
        check(qkv, pos, qk, out)
