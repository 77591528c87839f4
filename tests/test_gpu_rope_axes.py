"""rope_axes against the float64 oracle.

Bound: the fraction of a turn is rounded to fp32 (half a turn * 2^-24 * 2 pi =
3.2 * 2^-24 radians), sincospif is within 2 ulp (2^-23 at 1), the product and the
fused multiply-add round once each: under 8 * 2^-24 of |lo| + |hi| together; then
half a step of the output's type.
"""
import numpy as np
import pytest
import torch

from oracle import streaming as O

pytestmark = pytest.mark.gpu

STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def _check(got, x, pos, pairs):
    x = x.double().cpu().numpy()
    ref = O.rope_axes(x, pos.cpu().numpy(), pairs)
    size = np.zeros(x.shape)
    for lo, hi, _, _ in pairs:
        size[..., lo] = size[..., hi] = np.abs(x[..., lo]) + np.abs(x[..., hi])
    err = np.abs(got.double().cpu().numpy() - ref)
    step = STEP[got.dtype]
    assert (err <= np.abs(ref) * step + size * 8 * 2.0 ** -24 * (1 + step) + TINY[got.dtype]).all(), err.max()


@pytest.mark.parametrize("D,sections,layout", [
    (64, (32, 32), "block"), (64, (16, 24, 24), "block"), (64, (10, 26, 28), "block"), (64, (16, 8), "half"),
    (128, (32, 48, 48), "half"), (128, (22, 50, 56), "half"), (128, (64, 32), "block"), (16, (2, 2, 4, 8), "block"),
    (1024, (512, 512), "half"), (6, (2, 4), "half")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 1), (3, 5), (200, 3), (2500, 2)])
def test_rope_axes(gpu, D, sections, layout, dtype, T, H):
    """Every piece width (16 bytes down to one element), copied dims, one to four axes, far and negative positions."""
    from qvggt_amd import awq_inference_engine as E
    g = torch.Generator(device=gpu).manual_seed(D + T)
    x = torch.randn(T, H, D, generator=g, device=gpu).to(dtype)
    pos = torch.randint(-100, 2000000, (T, len(sections)), generator=g, device=gpu, dtype=torch.int32)
    plan = E.rope_axes_plan(D, sections, layout=layout, device=gpu)
    out = E.rope_axes(x, pos, plan)
    _check(out, x, pos, O.rope_pairs(sections, layout))
    rot = sum(sections)
    assert torch.equal(out[..., rot:], x[..., rot:])


def test_rope_axes_views_and_in_place(gpu):
    """The q and k heads inside a fused qkv buffer, rotated in place: the v heads stay, the bits are those of a copy."""
    from qvggt_amd import awq_inference_engine as E
    T, H, D = 333, 4, 64
    g = torch.Generator(device=gpu).manual_seed(0)
    qkv = torch.randn(T, 3 * H, D, generator=g, device=gpu).half()
    pos = torch.randint(0, 40, (T, 3), generator=g, device=gpu, dtype=torch.int32)
    plan = E.rope_axes_plan(D, (16, 24, 24), device=gpu)
    want = E.rope_axes(qkv[:, :2 * H].contiguous(), pos, plan)
    keep = qkv[:, 2 * H:].clone()
    got = E.rope_axes(qkv[:, :2 * H], pos, plan, out=qkv[:, :2 * H])
    assert torch.equal(got, want) and torch.equal(qkv[:, 2 * H:], keep)
    # odd strides and addresses: narrower pieces, the same bits
    wide = torch.randn(T * (2 * H * (D + 3)) + 1, generator=g, device=gpu).half()
    odd = wide[1:].view(T, 2 * H, D + 3)[..., :D]
    src = odd.clone()
    out = E.rope_axes(odd, pos, plan)
    assert torch.equal(out, E.rope_axes(src.contiguous(), pos, plan))
    # heads before tokens; dims not contiguous (copied)
    perm = src.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(E.rope_axes(perm, pos, plan), out)
    assert torch.equal(E.rope_axes(src.transpose(1, 2).contiguous().transpose(1, 2), pos, plan), out)


def test_rope_axes_other_stream_graph_and_empty(gpu):
    from qvggt_amd import awq_inference_engine as E
    g = torch.Generator(device=gpu).manual_seed(5)
    x = torch.randn(100, 8, 128, generator=g, device=gpu).bfloat16()
    pos = torch.randint(0, 4000, (100, 3), generator=g, device=gpu, dtype=torch.int32)
    plan = E.rope_axes_plan(128, (32, 48, 48), layout="half", device=gpu)
    want = E.rope_axes(x, pos, plan)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = E.rope_axes(x, pos, plan)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.rope_axes(x, pos, plan, out=out)
    for i in range(3):
        pos.add_(7)
        want = E.rope_axes(x, pos, plan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert E.rope_axes(x[:0], pos[:0], plan).shape == (0, 8, 128)


def test_rope_axes_non_finite_stays_in_its_pair(gpu):
    from qvggt_amd import awq_inference_engine as E
    x = torch.ones(4, 2, 64, device=gpu).half()
    x[1, 0, 3], x[2, 1, 40] = float("nan"), float("inf")
    pos = torch.full((4, 1), 5, dtype=torch.int32, device=gpu)
    out = E.rope_axes(x, pos, E.rope_axes_plan(64, (32,), device=gpu))
    bad = ~torch.isfinite(out)
    assert bad.nonzero().tolist() == [[1, 0, 3], [1, 0, 19], [2, 1, 40]]


@pytest.mark.parametrize("dtype,D,H,sections,layout", [(torch.float16, 64, 32, (16, 24, 24), "block"),
                                                       (torch.bfloat16, 128, 9, (40, 48), "half"),
                                                       (torch.float32, 64, 5, (32, 24), "block"),
                                                       (torch.float16, 512, 3, (512,), "half"),
                                                       (torch.float16, 64, 32, (10, 26, 28), "half"),
                                                       (torch.bfloat16, 64, 31, (12, 20, 20), "block"),
                                                       (torch.bfloat16, 128, 9, (22, 50, 56), "half"),
                                                       (torch.float16, 512, 3, (510,), "block"),
                                                       (torch.float16, 128, 1, (30, 34), "block"),
                                                       (torch.float32, 64, 5, (10, 26, 28), "half"),
                                                       (torch.float16, 256, 2, (6, 250), "half")])
def test_rope_axes_large(gpu, dtype, D, H, sections, layout):
    """Past 64 MB whole rows are taken, a lane each 8 dims, turned in registers or in LDS: the bits of the same tokens in small
    calls (in pieces), for a tensor of its own, inside a fused buffer and in place."""
    from qvggt_amd import awq_inference_engine as E
    T = (64 << 20) // (2 * H * D * torch.empty(0, dtype=dtype).element_size()) + 37
    g = torch.Generator(device=gpu).manual_seed(D)
    buf = torch.randn(T, H + 2, D, generator=g, device=gpu).to(dtype)
    x = buf[:, 1:-1]
    pos = torch.randint(-100, 100000, (T, len(sections)), generator=g, device=gpu, dtype=torch.int32)
    plan = E.rope_axes_plan(D, sections, layout=layout, device=gpu)
    want = torch.cat([E.rope_axes(x[i:i + 700], pos[i:i + 700], plan) for i in range(0, T, 700)])
    _check(want[:50], x[:50], pos[:50], O.rope_pairs(sections, layout))
    assert torch.equal(E.rope_axes(x, pos, plan), want)
    assert torch.equal(E.rope_axes(x.contiguous(), pos, plan), want)
    edge = buf[:, ::H + 1].clone()
    E.rope_axes(x, pos, plan, out=x)
    assert torch.equal(x, want) and torch.equal(buf[:, ::H + 1], edge)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [2, 4, 8, 16])
@pytest.mark.parametrize("T", [2047, 2048, 5000, 70001])
def test_rope_axes_one_piece_a_token(gpu, T, D, dtype):
    """One head whose pairs are one piece, several tokens to a workgroup: a tensor of its own, the first heads of a
    fused buffer in place (the others stay), heads before tokens (the head stride is the whole tensor)."""
    from qvggt_amd import awq_inference_engine as E
    g = torch.Generator(device=gpu).manual_seed(D + T)
    qkv = torch.randn(T, 3, D, generator=g, device=gpu).to(dtype)
    pos = torch.randint(-100, 100000, (T, 1), generator=g, device=gpu, dtype=torch.int32)
    plan = E.rope_axes_plan(D, (D,), device=gpu)
    x = qkv[:, :1].contiguous()
    out = E.rope_axes(x, pos, plan)
    _check(out, x, pos, O.rope_pairs((D,), "block"))
    rest = qkv[:, 1:].clone()
    assert torch.equal(E.rope_axes(qkv[:, :1], pos, plan, out=qkv[:, :1]), out)
    assert torch.equal(qkv[:, :1], out) and torch.equal(qkv[:, 1:], rest)
    before = x.view(1, T, D).transpose(0, 1)
    assert before.stride(1) == T * D
    into = torch.zeros(1, T, D, dtype=dtype, device=gpu).transpose(0, 1)
    assert torch.equal(E.rope_axes(before, pos, plan, out=into), out)


@pytest.mark.parametrize("D,sections", [(64, (16, 24, 24)), (30, (2, 4)), (16, (16,))])
def test_rope_axes_most_heads(gpu, D, sections):
    from qvggt_amd import awq_inference_engine as E
    g = torch.Generator(device=gpu).manual_seed(D)
    x = torch.randn(3, 4096, D, generator=g, device=gpu).half()
    pos = torch.randint(0, 5000, (3, len(sections)), generator=g, device=gpu, dtype=torch.int32)
    _check(E.rope_axes(x, pos, E.rope_axes_plan(D, sections, device=gpu)), x, pos, O.rope_pairs(sections, "block"))


@pytest.mark.parametrize("dtype,D,H,sections,layout,mb", [(torch.float16, 64, 8, (32, 32), "block", 260),
                                                          (torch.bfloat16, 128, 24, (128,), "half", 260),
                                                          (torch.float32, 64, 9, (32, 32), "half", 260),
                                                          (torch.float16, 128, 8, (64, 64), "block", 66),
                                                          (torch.float32, 64, 8, (16, 24, 24), "block", 66),
                                                          (torch.float16, 256, 8, (8, 64), "block", 66),
                                                          (torch.bfloat16, 512, 9, (8, 504), "half", 66),
                                                          (torch.float16, 512, 8, (510,), "block", 66),
                                                          (torch.bfloat16, 256, 8, (6, 250), "half", 66),
                                                          (torch.float16, 64, 7, (10, 26, 28), "block", 66),
                                                          (torch.float16, 64, 7, (16, 24, 24), "block", 66)])
def test_rope_axes_large_by_heads_and_pieces(gpu, dtype, D, H, sections, layout, mb):
    """Both sides of the rule that takes whole rows (heads, bytes, width of the pieces): the bits of the same tokens in
    small calls, inside a fused buffer and in place."""
    from qvggt_amd import awq_inference_engine as E
    T = (mb << 20) // (2 * H * D * torch.empty(0, dtype=dtype).element_size()) + 37
    g = torch.Generator(device=gpu).manual_seed(D + H)
    buf = torch.randn(T, H + 1, D, generator=g, device=gpu).to(dtype)
    x, edge = buf[:, 1:], buf[:, 0].clone()
    pos = torch.randint(-100, 100000, (T, len(sections)), generator=g, device=gpu, dtype=torch.int32)
    plan = E.rope_axes_plan(D, sections, layout=layout, device=gpu)
    want = torch.cat([E.rope_axes(x[i:i + 1500], pos[i:i + 1500], plan) for i in range(0, T, 1500)])
    _check(want[-50:], x[-50:], pos[-50:], O.rope_pairs(sections, layout))
    assert torch.equal(E.rope_axes(x, pos, plan), want)
    E.rope_axes(x, pos, plan, out=x)
    assert torch.equal(x, want) and torch.equal(buf[:, 0], edge)
