"""packed_attention against the float64 oracle: lengths around the tiles, frames, shared heads,
strides, what a query does not see, streams and graphs."""
import numpy as np
import pytest
import torch

from attention_bounds import close
from oracle import paged as P

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _qkv(gpu, seed, T, H, Hk, D, dtype, sharp=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return [(torch.randn(T, n, D, generator=g, device=gpu) * s).to(dtype) for n, s in ((H, sharp), (Hk, 1.0), (Hk, 1.0))]


def _check(out, q, k, v, lens, frame, scale=None):
    at = 0
    for n in lens:
        s = slice(at, at + n)
        if n:
            close(out[s], q[s], k[s], v[s], scale=scale, keep=P.seen_by_frame(n, frame), matched=True)
        at += n


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,Hk,frame", [
    ((1,), 1, 1, 1), ((1, 1, 1), 4, 2, 1), ((64,), 2, 2, 1), ((65, 63), 1, 1, 1), ((127, 0, 129), 3, 1, 1), ((200, 1, 77, 0), 8, 2, 1),
    ((300,), 5, 1, 1), ((31, 33, 32), 16, 2, 1), ((100, 257), 2, 1, 7), ((130, 64), 2, 2, 64), ((500,), 1, 1, 100), ((140, 3), 4, 4, None),
    ((513,), 2, 1, None), ((90, 260), 3, 3, 1000)])
def test_packed(gpu, lens, H, Hk, frame, D, dtype):
    from qvggt_amd import awq_inference_engine as E
    q, k, v = _qkv(gpu, sum(lens) + H, sum(lens), H, Hk, D, dtype)
    plan = E.packed_plan(lens, H, Hk, D, frame=frame, device=gpu)
    out = E.packed_attention(q, k, v, plan)
    assert out.shape == q.shape and torch.isfinite(out).all()
    _check(out, q, k, v, lens, frame)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,H,Hk,frame", [((300, 40, 257), 256, 256, 1), ((600,), 512, 256, 70), ((256, 513), 256, 256, None), ((129, 128, 1), 512, 256, 1)])
def test_packed_tiles_of_256_rows(gpu, lens, H, Hk, frame, dtype):
    """Many heads of 64: two blocks of 32 rows a wave."""
    from qvggt_amd import awq_inference_engine as E
    plan = E.packed_plan(lens, H, Hk, 64, frame=frame, device=gpu)
    assert plan.rows == 256
    q, k, v = _qkv(gpu, sum(lens) + H, sum(lens), H, Hk, 64, dtype, 2.0)
    out = E.packed_attention(q, k, v, plan)
    assert torch.isfinite(out).all()
    some = [0, 1, H // 2, H - 1]
    kv = [h // (H // Hk) for h in some]
    _check(out[:, some], q[:, some], k[:, kv], v[:, kv], lens, frame)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("sharp", [6.0, 40.0])
def test_packed_sharp_scores(gpu, D, dtype, sharp):
    """Scores up to hundreds: the running maximum moves between tiles."""
    from qvggt_amd import awq_inference_engine as E
    lens = (700, 90)
    q, k, v = _qkv(gpu, 5, sum(lens), 4, 2, D, dtype, sharp)
    plan = E.packed_plan(lens, 4, 2, D, device=gpu)
    _check(E.packed_attention(q, k, v, plan), q, k, v, lens, 1)
    _check(E.packed_attention(q, k, v, plan, scale=0.02), q, k, v, lens, 1, scale=0.02)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_packed_strides_and_rows_behind(gpu, D, dtype):
    """Views of a fused qkv buffer, strided outputs, tokens behind the last sequence."""
    from qvggt_amd import awq_inference_engine as E
    lens, H, Hk = (70, 150), 4, 2
    T = sum(lens) + 9
    g = torch.Generator(device=gpu).manual_seed(3)
    qkv = torch.randn(T, H + 2 * Hk, D, generator=g, device=gpu).to(dtype)
    qkv[sum(lens):] = float("nan")
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    plan = E.packed_plan(lens, H, Hk, D, device=gpu)
    out = E.packed_attention(q, k, v, plan)
    _check(out, q, k, v, lens, 1)
    assert not out[sum(lens):].any()
    wide = torch.full((T, 2 * H, D + 4), 7.0, device=gpu, dtype=dtype)
    assert E.packed_attention(q, k, v, plan, out=wide[:, ::2, :D]) is not None
    assert torch.equal(wide[:sum(lens), ::2, :D], out[:sum(lens)])
    assert (wide[sum(lens):] == 7).all() and (wide[:, 1::2] == 7).all() and (wide[..., D:] == 7).all()
    odd = torch.empty(T, H, D + 3, device=gpu, dtype=dtype)[..., :D].copy_(q)        # rows off 16 bytes: copied
    assert torch.equal(E.packed_attention(odd, k, v, plan)[:sum(lens)], out[:sum(lens)])
    empty = E.packed_plan((0, 0), H, Hk, D, device=gpu)
    assert E.packed_attention(q[:0], k[:0], v[:0], empty).shape == (0, H, D)
    assert not E.packed_attention(q, k, v, empty).any()
    assert E.packed_attention(q[:0], k[:0], v[:0], E.packed_plan((), H, Hk, D, device=gpu)).shape == (0, H, D)


@pytest.mark.parametrize("D,dtype,Hk", [(64, F16, 1), (128, BF16, 1), (128, F16, 1), (64, BF16, 1), (64, F16, 256), (64, BF16, 256)])
@pytest.mark.parametrize("frame", [1, 50])
def test_packed_non_finite_reaches_only_those_that_see_it(gpu, D, dtype, Hk, frame):
    """NaN and infinities of keys and values touch the queries that see them, and of values only their dims."""
    from qvggt_amd import awq_inference_engine as E
    lens, H = (300, 120), 2 * Hk
    q, k, v = _qkv(gpu, 7, sum(lens), H, Hk, D, dtype)
    plan = E.packed_plan(lens, H, Hk, D, frame=frame, device=gpu)
    clean = E.packed_attention(q, k, v, plan)
    bad = v.clone()
    bad[150, 0, 3], bad[201, 0, D - 1], bad[202, 0, D - 1], bad[290, 0, 17] = float("nan"), float("inf"), float("-inf"), float("inf")
    out = E.packed_attention(q, k, bad, plan)
    i = torch.arange(300, device=gpu)
    from_ = lambda t: (i // frame + 1) * frame > t
    want = clean[:300].clone()
    want[from_(150), :2, 3] = float("nan")
    want[from_(201), :2, D - 1] = float("inf")
    want[from_(202), :2, D - 1] = float("nan")
    want[from_(290), :2, 17] = float("inf")
    got = out[:300]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    ok = torch.isfinite(want)
    assert torch.equal(got[ok], want[ok])
    assert torch.equal(out[300:], clean[300:])
    bad = k.clone()
    bad[100] = float("nan")
    out = E.packed_attention(q, bad, v, plan)
    assert out[:300][from_(100)].isnan().all()
    assert torch.equal(out[:300][~from_(100)], clean[:300][~from_(100)]) and torch.equal(out[300:], clean[300:])


@pytest.mark.parametrize("D,dtype,Hk", [(64, F16, 1), (64, BF16, 1), (128, F16, 1), (128, BF16, 1), (64, F16, 256), (64, BF16, 256)])
@pytest.mark.parametrize("frame", [1, 50, None])
def test_packed_infinities_of_the_first_tokens(gpu, D, dtype, Hk, frame):
    """In the first tile an infinity reaches those that see it as one, too; two of unlike signs as NaN."""
    from qvggt_amd import awq_inference_engine as E
    lens, H = (300, 120), 2 * Hk
    q, k, v = _qkv(gpu, 7, sum(lens), H, Hk, D, dtype, 0.25)
    plan = E.packed_plan(lens, H, Hk, D, frame=frame, device=gpu)
    assert plan.rows == (256 if Hk == 256 else 128)
    clean = E.packed_attention(q, k, v, plan)
    bad, want, inf = v.clone(), clean.clone(), float("inf")
    i = torch.arange(300, device=gpu)
    from_ = lambda t: ((i // frame + 1) * frame if frame else torch.full_like(i, 300)) > t
    for t, dim, x in ((0, 0, inf), (0, 1, -inf), (40, 2, inf), (40, 3, -inf), (63, 4, inf), (64, 5, -inf), (127, 6, inf)):
        bad[t, 0, dim] = x
        want[:300][from_(t), :2, dim] = x
    bad[0, 0, 7], bad[40, 0, 7] = inf, -inf
    want[:300][from_(0), :2, 7] = inf
    want[:300][from_(40), :2, 7] = float("nan")
    out = E.packed_attention(q, k, bad, plan)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
    ok = ~want.isnan()
    assert torch.equal(out[ok], want[ok])


def test_packed_long_sequence(gpu):
    """A longer one, some heads and rows of it against the definition."""
    from qvggt_amd import awq_inference_engine as E
    lens, H, Hk, D = (5000, 3), 8, 2, 128
    q, k, v = _qkv(gpu, 9, sum(lens), H, Hk, D, BF16)
    out = E.packed_attention(q, k, v, E.packed_plan(lens, H, Hk, D, device=gpu))
    for at in (0, 63, 64, 2047, 4990, 4999):
        close(out[at:at + 1], q[at:at + 1], k[:at + 1], v[:at + 1], matched=True)
    close(out[5000:], q[5000:], k[5000:], v[5000:], keep=P.seen_by_frame(3, 1), matched=True)


def test_packed_streams_and_graphs(gpu):
    """On another stream and replayed from a graph: the same bits."""
    from qvggt_amd import awq_inference_engine as E
    lens, H, Hk, D = (190, 33), 4, 1, 64
    q, k, v = _qkv(gpu, 11, sum(lens), H, Hk, D, F16)
    plan = E.packed_plan(lens, H, Hk, D, device=gpu)
    want = E.packed_attention(q, k, v, plan)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = E.packed_attention(q, k, v, plan)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = E.packed_attention(q, k, v, plan)
    for i in range(3):
        q.mul_(-1.0)
        want = E.packed_attention(q, k, v, plan)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_packed_a_tile_outside_the_tokens_is_left_out(gpu):
    """The C entry takes tiles from the device: ones that do not fit are skipped."""
    from qvggt_amd import awq_inference_engine as E
    q, k, v = _qkv(gpu, 13, 40, 2, 1, 64, F16)
    plan = E.packed_plan((40,), 2, 1, 64, device=gpu)
    want = E.packed_attention(q, k, v, plan)
    bad = torch.tensor([[0, 41, 0, 0], [-1, 40, 0, 0], [10, 31, 0, 0], [0, 40, 80, 0], [0, 40, -128, 0], [0, 0, 0, 0], [0, -5, 0, 0],
                        [2 ** 31 - 1, 40, 0, 0], [0, 2 ** 31 - 1, 0, 0]], dtype=torch.int32, device=gpu)
    out = torch.full_like(q, 3.0)
    E.packed_attention(q, k, v, plan._replace(tiles=bad), out=out)
    assert (out == 3).all()
    E.packed_attention(q, k, v, plan._replace(tiles=torch.cat([bad, plan.tiles])), out=out)
    assert torch.equal(out, want)
