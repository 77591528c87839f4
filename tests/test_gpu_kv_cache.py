"""Int8KVCache's append and values, bit for bit against the oracle (float64 and whole numbers).

Every scale has four significant bits and every input at most 11, so codes,
scales and values are exact in the kernels: nothing here has a tolerance.
"""
import numpy as np
import pytest
import torch

from oracle import streaming as O

pytestmark = pytest.mark.gpu


class Both:
    """The cache and one oracle per (sequence, tensor)."""

    def __init__(self, gpu, B, H, D, capacity):
        from qvggt_amd.kv_cache import Int8KVCache
        self.cache = Int8KVCache(B, H, D, capacity, device=gpu)
        self.ref = [[O.Cache(self.cache.capacity, H, D) for _ in range(2)] for _ in range(B)]

    def append(self, k, v, counts=None, start=None, call=None):
        dev = self.cache.lens.device
        t = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32, device=dev)
        (call or self.cache.append)(k, v, counts=t(counts), start=t(start))
        for b, refs in enumerate(self.ref):
            n = k.shape[1] if counts is None else counts[b]
            for r, x in zip(refs, (k, v)):
                r.append(x[b, :n].double().cpu().numpy(), None if start is None else start[b])

    def check(self):
        assert self.cache.lens.tolist() == [r[0].len for r in self.ref]
        kc, ks, vc, vs, _ = (t.cpu().numpy() for t in self.cache.save_codes())
        got = [t.cpu().numpy() for t in self.cache.values()]
        for b, refs in enumerate(self.ref):
            n = refs[0].len
            for r, c, s, x in zip(refs, (kc[b], vc[b]), (ks[b], vs[b]), got):
                nb = -(-n // O.BLOCK)
                np.testing.assert_array_equal(s[:nb], r.scales[:nb])
                live = np.repeat(~np.isnan(r.scales), O.BLOCK, 0)[:n]
                np.testing.assert_array_equal(c[:n][live], r.codes[:n][live])
                np.testing.assert_array_equal(x[b, :n], r.values())
                assert not x[b, n:].any()


def _kv(gpu, g, B, n, H, D, dtype, size=1.0):
    chan = torch.exp(torch.randn(H, D, generator=g, device=gpu))
    return [(torch.randn(B, n, H, D, generator=g, device=gpu) * chan * size).to(dtype) for _ in range(2)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_in_pieces(gpu, D, dtype):
    """One token, a few, up to a block's end, over one, many blocks: growing scales in half-filled blocks."""
    both = Both(gpu, 2, 3, D, 700)
    g = torch.Generator(device=gpu).manual_seed(D)
    for i, n in enumerate((1, 1, 5, 57, 64, 1, 62, 2, 190, 0, 63, 65)):
        both.append(*_kv(gpu, g, 2, n, 3, D, dtype, 1.0 + 0.4 * (i % 3)))
        both.check()


def test_single_tokens_grow_the_scale(gpu):
    both = Both(gpu, 1, 2, 64, 64)
    g = torch.Generator(device=gpu).manual_seed(3)
    for i in range(64):
        both.append(*_kv(gpu, g, 1, 1, 2, 64, torch.float16, 1.02 ** i))
        both.check()


@pytest.mark.parametrize("D", [64, 128])
def test_ragged_counts_and_start(gpu, D):
    """Padding is not read (NaN there), sequences of different lengths, a call for none; falling back to an earlier start."""
    both = Both(gpu, 4, 2, D, 320)
    g = torch.Generator(device=gpu).manual_seed(D + 1)
    for counts, start in (([70, 0, 1, 130], None), ([3, 64, 63, 100], None), ([10, 20, 30, 40], [64, 0, 10, 200]),
                          ([0, 0, 0, 0], [60, 20, 1, 0]), ([130, 1, 100, 128], None)):
        k, v = _kv(gpu, g, 4, 130, 2, D, torch.float16)
        for b, c in enumerate(counts):
            k[b, c:], v[b, c:] = float("nan"), float("inf")
        both.append(k, v, counts, start)
        both.check()
    both.cache.reset()
    assert not both.cache.values()[0].any()


def test_capacity_stops_the_sequence(gpu):
    both = Both(gpu, 2, 1, 64, 128)
    g = torch.Generator(device=gpu).manual_seed(4)
    both.append(*_kv(gpu, g, 2, 100, 1, 64, torch.float16))
    both.append(*_kv(gpu, g, 2, 60, 1, 64, torch.float16), [60, 5])
    both.check()
    assert both.cache.lens.tolist() == [128, 105]
    both.append(*_kv(gpu, g, 2, 7, 1, 64, torch.float16))
    both.check()
    # a start or count outside the cache is drawn into it
    one = torch.tensor([-5, 1000], dtype=torch.int32, device=gpu)
    k, v = _kv(gpu, g, 2, 3, 1, 64, torch.float16)
    both.cache.append(k, v, start=one, counts=torch.tensor([-1, 100], dtype=torch.int32, device=gpu))
    assert both.cache.lens.tolist() == [0, 128]


@pytest.mark.parametrize("dtype,peak", [(torch.float16, 65504.0), (torch.bfloat16, 3e38), (torch.bfloat16, 1e-38),
                                        (torch.float16, 2.0 ** -24), (torch.float16, 0.0)])
def test_extreme_sizes(gpu, dtype, peak):
    """The largest and smallest numbers, zero blocks, ties of every code."""
    both = Both(gpu, 1, 2, 64, 128)
    g = torch.Generator(device=gpu).manual_seed(9)
    k = ((torch.rand(1, 70, 2, 64, generator=g, device=gpu) * 2 - 1) * peak).to(dtype)
    k[0, 0, 0, 0] = peak
    both.append(k, -k)
    both.check()
    ties = ((torch.arange(64 * 64, device=gpu) % 255 - 127) / 2).view(1, 64, 1, 64).expand(1, 64, 2, 64).to(dtype)
    both.append(ties.contiguous(), ties.contiguous() * 2, start=[64])
    both.check()


def test_non_finite_marks_its_block_and_head(gpu):
    both = Both(gpu, 1, 3, 64, 256)
    g = torch.Generator(device=gpu).manual_seed(11)
    k, v = _kv(gpu, g, 1, 100, 3, 64, torch.float16)
    k[0, 70, 1, 5], v[0, 3, 2, 0] = float("nan"), float("-inf")
    both.append(k, v)
    both.check()
    both.append(*_kv(gpu, g, 1, 100, 3, 64, torch.float16))      # the marked half-filled block stays marked
    both.check()
    kk, vv = both.cache.values(200)
    assert kk.isnan().any(3)[0].nonzero().tolist() == [[t, 1] for t in range(64, 128)]
    assert vv.isnan().any(3)[0].nonzero().tolist() == [[t, 2] for t in range(64)]
    both.append(*_kv(gpu, g, 1, 50, 3, 64, torch.float16), start=[0])   # begun again
    both.check()
    assert torch.isfinite(both.cache.values(50)[1]).all()


def test_strided_inputs(gpu):
    """The k and v heads inside a fused qkv buffer, heads before tokens, and rows that have to be copied."""
    g = torch.Generator(device=gpu).manual_seed(12)
    H, D = 3, 64
    qkv = torch.randn(2, 90, 3 * H, D, generator=g, device=gpu).half()
    forms = [qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]]
    perm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in forms]
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in forms]
    for k, v in (forms, perm, odd, (forms[0], perm[1])):
        both = Both(gpu, 2, H, D, 128)
        both.append(k, v)
        both.check()
    one = qkv[:1, :, H:2 * H].expand(2, 90, H, D)                # one prompt for all sequences
    both = Both(gpu, 2, H, D, 128)
    both.append(one, one)
    both.check()


@pytest.mark.parametrize("D", [64, 128])
def test_values_ranges_and_types(gpu, D):
    both = Both(gpu, 3, 2, D, 300)
    g = torch.Generator(device=gpu).manual_seed(13)
    both.append(*_kv(gpu, g, 3, 250, 2, D, torch.float16), [250, 64, 7])
    full = both.cache.values()
    for n, first in ((1, [0, 5, 249]), (64, [64, 0, 1]), (130, [63, 300, 6]), (500, [0, 1, 319]), (70, [-3, 4000, 0])):
        got = both.cache.values(n, torch.tensor(first, dtype=torch.int32, device=gpu))
        for f, x in zip(full, got):
            for b, at in enumerate(min(max(a, 0), both.cache.capacity) for a in first):
                want = torch.nn.functional.pad(f[b], (0, 0, 0, 0, 0, n))[at:at + n]
                assert torch.equal(x[b], want)
    for dtype in (torch.float16, torch.bfloat16):
        for f, x in zip(full, both.cache.values(dtype=dtype)):
            assert torch.equal(x, f.to(dtype))
    assert torch.equal(full[0], both.cache.values(dtype=torch.float16)[0].float())    # fp16 holds them
    assert both.cache.values(0)[0].shape == (3, 0, 2, D)


def test_save_and_load(gpu):
    from qvggt_amd.kv_cache import Int8KVCache
    both = Both(gpu, 2, 3, 128, 200)
    g = torch.Generator(device=gpu).manual_seed(14)
    both.append(*_kv(gpu, g, 2, 150, 3, 128, torch.bfloat16), [150, 33])
    other = Int8KVCache(2, 3, 128, 500, device=gpu)
    other.load_codes(*both.cache.save_codes())
    both.cache = other
    for r in sum(both.ref, []):
        r.codes, r.scales = np.pad(r.codes, ((0, 256), (0, 0), (0, 0))), np.pad(r.scales, ((0, 4), (0, 0)))
    both.check()
    both.append(*_kv(gpu, g, 2, 77, 3, 128, torch.bfloat16))
    both.check()
    k_codes, k_scales, v_codes, v_scales, lens = other.save_codes()
    for bad in ((k_codes[:, :10], k_scales, v_codes, v_scales, lens), (k_codes, k_scales * 1.03, v_codes, v_scales, lens),
                (k_codes, -1 - k_scales, v_codes, v_scales, lens), (k_codes, k_scales, v_codes, v_scales, lens + 9999),
                (k_codes, k_scales, v_codes.fill_(-128), v_scales, lens)):
        with pytest.raises(RuntimeError, match="load_codes"):
            other.load_codes(*bad)


def test_append_in_a_graph_and_on_another_stream(gpu):
    """A replayed append goes on from the lengths that it finds; eager calls between the replays."""
    both = Both(gpu, 2, 2, 64, 400)
    g = torch.Generator(device=gpu).manual_seed(15)
    k, v = _kv(gpu, g, 2, 3, 2, 64, torch.float16)
    both.append(k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both.cache.append(k, v)
    for i in range(5):
        for t, fresh in zip((k, v), _kv(gpu, g, 2, 3, 2, 64, torch.float16, 1.0 + i)):
            t.copy_(fresh)
        both.append(k, v, call=lambda *a, **kw: graph.replay())
        both.check()
        both.append(*_kv(gpu, g, 2, 30, 2, 64, torch.float16))
        both.check()
    st = torch.cuda.Stream()
    k, v = _kv(gpu, g, 2, 50, 2, 64, torch.float16)
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        both.append(k, v)
    torch.cuda.current_stream().wait_stream(st)
    both.check()


@pytest.mark.parametrize("B,H,n", [(3, 2, 1), (2, 5, 700), (4, 1, 65)])
def test_lens_advance_by_themselves(gpu, B, H, n):
    """start left out, or lens itself: the length moves on once all of a sequence's workgroups have read it,
    call after call; the same contents as with a start of its own."""
    from qvggt_amd.kv_cache import Int8KVCache
    g = torch.Generator(device=gpu).manual_seed(n)
    a, b, c = (Int8KVCache(B, H, 64, 3000, device=gpu) for _ in range(3))
    at = torch.zeros(B, dtype=torch.int32, device=gpu)
    for i in range(4):
        k, v = _kv(gpu, g, B, n, H, 64, torch.float16)
        counts = torch.randint(0, n + 1, (B,), generator=g, device=gpu, dtype=torch.int32)
        a.append(k, v, counts=counts)
        b.append(k, v, counts=counts, start=b.lens)
        c.append(k, v, counts=counts, start=at)
        at = at + counts
        assert a.lens.tolist() == b.lens.tolist() == c.lens.tolist() == at.tolist()
    for x, y, z in zip(a.values(), b.values(), c.values()):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("own_start", [False, True])
def test_counts_are_lens(gpu, own_start):
    """lens itself as the counts: written once every workgroup of the sequence has read it."""
    from qvggt_amd.kv_cache import Int8KVCache
    g = torch.Generator(device=gpu).manual_seed(5)
    for _ in range(4):
        a, b = (Int8KVCache(3, 6, 64, 4000, device=gpu) for _ in range(2))
        for c in (a, b):
            c.lens.copy_(torch.tensor([1900, 0, 70], dtype=torch.int32))
        k, v = _kv(gpu, g, 3, 2000, 6, 64, torch.float16)
        start = torch.tensor([5, 64, 0], dtype=torch.int32, device=gpu) if own_start else None
        a.append(k, v, counts=a.lens, start=start)
        b.append(k, v, counts=b.lens.clone(), start=start)
        assert a.lens.tolist() == b.lens.tolist() == ([1905, 64, 70] if own_start else [3800, 0, 140])
        n = a.lens.max().item()
        for x, y in zip(a.values(n), b.values(n)):
            assert torch.equal(x, y)


def test_many_workgroups_without_tokens(gpu):
    """Sequences of a few tokens, some of none, in a launch for thousands, lens as the start: workgroups
    that find nothing to do read the start too before it moves."""
    from qvggt_amd.kv_cache import Int8KVCache
    g = torch.Generator(device=gpu).manual_seed(8)
    a, b = (Int8KVCache(7, 9, 64, 6400, device=gpu) for _ in range(2))
    at = torch.zeros(7, dtype=torch.int32, device=gpu)
    for i in range(6):
        k, v = _kv(gpu, g, 7, 5000, 9, 64, torch.float16)
        counts = torch.tensor([0, 1, 63, 64, 65, 130, 2 * i], dtype=torch.int32, device=gpu)
        a.append(k, v, counts=counts)
        b.append(k, v, counts=counts, start=at)
        at = at + counts
        assert a.lens.tolist() == b.lens.tolist() == at.tolist()
    for x, y in zip(a.values(800), b.values(800)):
        assert torch.equal(x, y)
