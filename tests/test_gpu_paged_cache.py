"""PagedKVCache: contents bit for bit and attention within its bounds against the float64 oracle."""
import numpy as np
import pytest
import torch

from attention_bounds import close, received_close
from oracle import paged as P

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _i32(gpu, a):
    return None if a is None else torch.tensor(a, dtype=torch.int32, device=gpu)


class Both:
    """A cache whose pages are given out in any order, and one oracle per sequence."""

    def __init__(self, gpu, B, Hk, D, capacity, page, dtype, track=True, seed=0, own=False):
        from qvggt_amd.kv_cache import PagedKVCache
        self.gpu, self.g = gpu, torch.Generator(device=gpu).manual_seed(seed)
        slots = -(-capacity // page)
        self.cache = PagedKVCache(B, Hk, D, capacity, page=page, pages=None if own else B * slots + 3, dtype=dtype, track=track, device=gpu)
        if not own:
            self.cache.table.copy_(torch.randperm(B * slots + 3, generator=self.g, device=gpu)[:B * slots].view(B, slots))
        self.cache.k_pages.fill_(float("nan"))       # what is not written may hold anything
        self.cache.v_pages.fill_(float("nan"))
        self.ref = [P.Sequence(self.cache.capacity, Hk, D) for _ in range(B)]
        for r in self.ref:
            r.rows.fill(np.nan)

    def rand(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.gpu).to(self.cache.dtype)

    def kv(self, *lead):
        c = self.cache
        return self.rand(*lead, c.kv_heads, c.head_dim), self.rand(*lead, c.kv_heads, c.head_dim)

    def append(self, n, counts=None, start=None, call=None):
        c = self.cache
        k, v = self.kv(c.batch, n)
        if counts is not None:
            for b, m in enumerate(counts):
                k[b, m:], v[b, m:] = float("nan"), float("inf")
        (call or c.append)(k, v, counts=_i32(self.gpu, counts), start=_i32(self.gpu, start))
        for b, r in enumerate(self.ref):
            m = n if counts is None else counts[b]
            r.append(k[b, :m].double().cpu().numpy(), v[b, :m].double().cpu().numpy(), None if start is None else start[b])

    def rows(self, b, n):
        """Keys and values of the first n slots of a sequence, (n, Hk, D); those without a page are any."""
        c = self.cache
        pages = c.table[b].long().clamp(0, c.pages - 1)
        return [x[pages].transpose(1, 2).reshape(-1, c.kv_heads, c.head_dim)[:n] for x in (c.k_pages, c.v_pages)]

    def check(self):
        c = self.cache
        assert c.lens.tolist() == [r.len for r in self.ref]
        for b, r in enumerate(self.ref):
            for got, want in zip(self.rows(b, r.len), r.rows):
                np.testing.assert_array_equal(got.double().cpu().numpy(), want[:r.len])
            if c.weights is not None:
                np.testing.assert_array_equal(c.positions[b, :, :r.len].cpu().numpy(), r.positions[:, :r.len])
                np.testing.assert_array_equal(c.weights[b, :, :r.len].cpu().numpy(), r.weights[:, :r.len].astype(np.float32))
        if c.weights is not None:
            assert c.evicted.tolist() == [r.evicted for r in self.ref]

    def attend(self, q, **kw):
        """Outputs, and with collect what was received, within their bounds."""
        c, n = self.cache, q.shape[1]
        before = c.weights.clone() if kw.get("collect") else None
        if before is not None:
            c.weights.zero_()
        out = c.attention(q, **kw)
        counts = [n] * c.batch if kw.get("counts") is None else kw["counts"].tolist()
        for b, (r, m) in enumerate(zip(self.ref, counts)):
            k, v = self.rows(b, r.len)
            there = np.repeat(((c.table[b] >= 0) & (c.table[b] < c.pages)).cpu().numpy(), c.page)[:r.len]
            keep = np.broadcast_to(there, (m, r.len))
            if kw.get("causal"):
                keep = keep & (np.arange(r.len)[None] <= (r.len - m + np.arange(m))[:, None])
            assert torch.isfinite(out[b, :m]).all()
            if r.len:
                k, v = (torch.where(torch.from_numpy(there.copy()).to(self.gpu)[:, None, None], x, 0) for x in (k, v))
                close(out[b, :m], q[b, :m], k, v, scale=kw.get("scale"), keep=keep)
            else:
                assert not out[b, :m].any()
            if before is not None:
                if r.len and m:
                    received_close(c.weights[b, :, :r.len], q[b, :m], k, scale=kw.get("scale"), keep=keep)
                assert not c.weights[b, :, r.len:].any()
        if before is not None:
            c.weights.add_(before)
        return out


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_append_in_pieces(gpu, page, D, dtype):
    both = Both(gpu, 3, 2, D, 600, page, dtype)
    for n in (1, 1, 14, 48, 0, 63, 200, 2):
        both.append(n)
        both.check()


def test_append_counts_start_and_capacity(gpu):
    both = Both(gpu, 4, 3, 64, 320, 32, F16)
    for counts, start in (([70, 0, 1, 130], None), ([3, 64, 63, 100], None), ([10, 20, 30, 40], [64, 0, 10, 200]),
                          ([0, 0, 0, 0], [60, 20, 1, 0]), ([130, 1, 100, 128], None), ([130, 130, 130, 130], [0, 300, 189, 190])):
        both.append(130, counts, start)
        both.check()
    both.cache.reset()
    assert not both.cache.lens.any() and not both.cache.evicted.any()
    k, v = both.kv(4, 3)
    # a start or count outside the cache is drawn into it
    both.cache.append(k, v, start=_i32(gpu, [-5, 1000, 320, 318]), counts=_i32(gpu, [-1, 100, 3, 3]))
    assert both.cache.lens.tolist() == [0, 320, 320, 320]


@pytest.mark.parametrize("how", ["padded", "packed", "graph"])
def test_append_keeps_the_account_in_front_of_start(gpu, how):
    """What a program wrote there itself (a restored cache, a beginning of another sequence) stays, whatever lens says;
    the new tokens' own, and nothing behind them, are written."""
    from qvggt_amd import awq_inference_engine as E
    both = Both(gpu, 6, 2, 64, 256, 16, F16)
    c, n = both.cache, (3, 1, 0, 40, 10, 7)
    lens, start, gone = [0, 5, 100, 0, 200, 256], [200, 30, 90, 64, 250, 300], [0, 7, 1000, 3, 0, 9]
    given = torch.rand(c.weights.shape, generator=both.g, device=gpu)
    pos = torch.randint(0, 1 << 20, c.positions.shape, generator=both.g, device=gpu, dtype=torch.int32)
    k, v = both.kv(sum(n)) if how == "packed" else both.kv(6, 40)
    plan = E.packed_plan(n, 2, 2, 64, device=gpu) if how == "packed" else None
    counts, begin = None if plan else _i32(gpu, n), _i32(gpu, start)

    def put():
        c.lens.copy_(_i32(gpu, lens))
        c.evicted.copy_(_i32(gpu, gone))
        c.weights.copy_(given)
        c.positions.copy_(pos)

    call = lambda: c.append(k, v, counts=counts, start=begin, plan=plan)
    if how == "graph":
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=s):
            call()
        call = graph.replay
    for _ in range(3):
        put()
        call()
        torch.cuda.synchronize()
        want_w, want_p = given.clone(), pos.clone()
        for b in range(6):
            s, e = min(start[b], 256), min(start[b] + n[b], 256)
            want_w[b, :, s:e] = 0
            want_p[b, :, s:e] = torch.arange(s, e, device=gpu, dtype=torch.int32) + gone[b]
            assert c.lens[b] == e
        assert torch.equal(c.weights, want_w) and torch.equal(c.positions, want_p)


@pytest.mark.parametrize("D,dtype,track", [(64, BF16, False), (128, F16, True)])
def test_append_packed(gpu, D, dtype, track):
    """Packed tokens, of a strided buffer with rows behind them."""
    from qvggt_amd import awq_inference_engine as E
    both = Both(gpu, 4, 2, D, 300, 16, dtype, track=track)
    for lens in ((5, 0, 130, 17), (1, 1, 1, 1), (100, 50, 2, 0), (0, 0, 0, 0), (250, 3, 2, 100)):
        plan = E.packed_plan(lens, 4, 2, D, device=gpu)
        kv = both.rand(sum(lens) + 4, 5, D)
        k, v = kv[:, :2], kv[:, 3:]
        both.cache.append(k, v, plan=plan)
        for r, a, n in zip(both.ref, np.cumsum((0,) + lens), lens):
            r.append(*(x[a:a + n].double().cpu().numpy() for x in (k, v)))
        both.check()


def test_append_without_a_page_is_dropped(gpu):
    both = Both(gpu, 2, 1, 64, 128, 32, F16)
    both.cache.table[0, 1] = -1
    both.cache.table[1, 0] = both.cache.pages
    before = both.cache.k_pages.clone()
    k, v = both.kv(2, 100)
    both.cache.append(k, v)
    got = both.cache.k_pages
    written = [(0, 0), (0, 2), (0, 3), (1, 1), (1, 2), (1, 3)]
    for b, i in written:
        n = min(32, 100 - 32 * i)
        assert torch.equal(got[both.cache.table[b, i].long(), 0, :n], k[b, 32 * i:32 * i + n, 0])
    rest = torch.ones(both.cache.pages, dtype=torch.bool, device=gpu)
    rest[[int(both.cache.table[b, i]) for b, i in written]] = False
    assert got[rest].isnan().all() and before.isnan().all()
    assert both.cache.lens.tolist() == [100, 100]


# --------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("n,H,Hk,causal", [(1, 1, 1, False), (1, 8, 2, True), (3, 5, 1, True), (7, 4, 1, False), (32, 2, 2, True), (9, 8, 2, True),
                                           (60, 3, 1, True), (130, 2, 2, True), (150, 2, 1, False)])
def test_attention(gpu, n, H, Hk, causal, page, D, dtype):
    """Few and many queries, lengths around tiles and pages, with what is received."""
    both = Both(gpu, 4, Hk, D, 700, page, dtype, seed=n)
    both.append(700, [n, 64 + n, 333, 700])
    both.attend(both.rand(4, n, H, D), causal=causal, collect=True)


@pytest.mark.parametrize("n,H,Hk", [(1, 4, 1), (40, 2, 1)])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_attention_lengths_counts_and_missing_pages(gpu, n, H, Hk, D, dtype):
    both = Both(gpu, 6, Hk, D, 400, 16, dtype)
    both.append(400, [0, 1, 15, 17, 64, 400])
    q = both.rand(6, n, H, D)
    both.attend(q, collect=True)
    both.attend(q, causal=True, collect=True)                # queries before the first token see nothing
    both.cache.table[5, 3] = -1
    both.cache.table[5, 20] = 1 << 30
    both.cache.table[4, :] = -7
    both.attend(q, collect=True)
    both.attend(q, causal=True, collect=True, scale=0.3)
    counts = _i32(gpu, [n, 0, n // 2, 1, n, 0])
    q2 = q.clone()
    for b, c in enumerate(counts.tolist()):
        q2[b, c:] = float("nan")
    out = torch.full_like(q, 5.0)
    both.attend(q2, causal=True, counts=counts, collect=True, out=out)
    for b, c in enumerate(counts.tolist()):
        assert (out[b, c:] == 5).all()
    fresh = both.cache.attention(q2, causal=True, counts=counts)
    for b, c in enumerate(counts.tolist()):
        assert torch.equal(fresh[b, :c], out[b, :c]) and not fresh[b, c:].any()
    with_lens = both.cache.lens.clone()
    both.cache.lens.copy_(_i32(gpu, [-3, 1, 15, 17, 64, 100000]))       # drawn into 0 .. capacity
    got = both.cache.attention(q)
    both.cache.lens.copy_(with_lens)
    assert torch.equal(got, both.cache.attention(q))


@pytest.mark.parametrize("n,H,Hk,D,dtype", [(1, 8, 2, 128, BF16), (1, 4, 4, 64, F16), (5, 4, 1, 128, F16), (50, 2, 1, 64, BF16),
                                           (70, 4, 2, 128, BF16)])
def test_attention_split_keys(gpu, n, H, Hk, D, dtype):
    """Many keys of few heads: split and joined; any hint of the length gives the result; repeatable."""
    from qvggt_amd import _lib
    both = Both(gpu, 2, Hk, D, 9000, 64, dtype)
    both.append(9000, [9000, 2500])
    assert _lib.load().qv_paged_attention_workspace(0, 2, n, H, Hk, D, 9000, 9024) > 0
    q = both.rand(2, n, H, D) * 3
    out = both.attend(q, causal=True, collect=True)
    assert torch.equal(out, both.cache.attention(q, causal=True))
    for longest in (0, 1, 700, 100000):
        both.attend(q, causal=True, longest=longest, collect=True)


@pytest.mark.parametrize("n,H,Hk", [(4, 4, 1), (60, 2, 1)])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_attention_non_finite(gpu, n, H, Hk, D, dtype):
    """A causal query is touched by what it sees, and of values in their dims only."""
    both = Both(gpu, 1, Hk, D, 500, 32, dtype)
    both.append(500)
    q = both.rand(1, n, H, D)
    clean = both.cache.attention(q, causal=True)
    _, v = both.rows(0, 500)
    at = lambda s: (both.cache.table[0, s // 32].long(), 0, s % 32)
    s = 500 - n + 2                                          # the third query's own token
    both.cache.v_pages[at(s)][5] = float("nan")
    both.cache.v_pages[at(s + 1)][D - 1] = float("-inf")
    out = both.cache.attention(q, causal=True)
    want = clean.clone()
    want[:, 2:, :, 5] = float("nan")
    want[:, 3:, :, D - 1] = float("-inf")
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
    ok = torch.isfinite(want)
    assert torch.equal(out[ok], want[ok])


@pytest.mark.parametrize("n,H,Hk", [(1, 1, 1), (4, 4, 1), (3, 2, 2), (32, 1, 1), (60, 2, 1), (130, 1, 1)])
@pytest.mark.parametrize("D,dtype", [(64, F16), (64, BF16), (128, F16), (128, BF16)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("tokens", [500, 9000])
def test_attention_infinite_values_anywhere(gpu, tokens, causal, D, dtype, n, H, Hk):
    """An infinity that all queries see is one in its dim, in the first tile of a wave, a share or a piece as well; two
    of unlike signs are NaN.  (9000 tokens: shares of 256 slots.)"""
    both = Both(gpu, 1, Hk, D, tokens, 32, dtype)
    both.append(tokens)
    q = both.rand(1, n, H, D) / 4                            # even weights: none comes to 0 in 32 bits
    clean = both.attend(q, causal=causal)
    at = lambda s: (both.cache.table[0, s // 32].long(), slice(None), s % 32)
    inf, want = float("inf"), clean.clone()
    slots = [0, 40, 64, 127, 128, 255, tokens - n] + ([256, 300, 4096, 4100, 8191] if tokens > 500 else [])
    for i, s in enumerate(slots):
        both.cache.v_pages[at(s)][:, i] = inf if i % 2 else -inf
        want[..., i] = inf if i % 2 else -inf
    both.cache.v_pages[at(0)][:, 40], both.cache.v_pages[at(33)][:, 40] = inf, -inf
    want[..., 40] = float("nan")
    both.cache.v_pages[at(1)][:, 41] = float("nan")
    want[..., 41] = float("nan")
    out = both.cache.attention(q, causal=causal)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
    ok = ~want.isnan()
    assert torch.equal(out[ok], want[ok])


def test_shared_pages(gpu):
    """Two sequences read the pages of one beginning."""
    both = Both(gpu, 2, 2, 64, 256, 64, F16)
    both.append(128, [128, 0])
    both.cache.table[1, :2] = both.cache.table[0, :2]
    both.ref[1].rows[:, :128] = both.ref[0].rows[:, :128]
    both.append(60, [10, 60], start=[128, 128])              # takes what the pages hold
    both.check()
    both.attend(both.rand(2, 1, 4, 64), collect=True)


@pytest.mark.parametrize("B", [129, 300])
@pytest.mark.parametrize("D,dtype,H,Hk", [(64, F16, 4, 2), (128, BF16, 2, 2)])
def test_attention_of_many_sequences(gpu, B, D, dtype, H, Hk):
    """More sequences than threads look for a share's first one; empty ones and ones without queries among them."""
    both = Both(gpu, B, Hk, D, 96, 16, dtype)
    lens = [(37 * b) % 97 for b in range(B)]
    both.append(96, lens)
    q = both.rand(B, 3, H, D)
    counts = _i32(gpu, [(b * 7) % 4 for b in range(B)])
    for longest in (96, 100000):                             # whole sequences; shares of all
        both.attend(q, causal=True, longest=longest, collect=True)
        both.attend(q, counts=counts, longest=longest, collect=True)


@pytest.mark.parametrize("B", [3, 64, 65, 300])
@pytest.mark.parametrize("D,dtype,H,Hk", [(64, F16, 4, 1), (128, BF16, 1, 1)])
def test_attention_of_many_rows_and_sequences(gpu, B, D, dtype, H, Hk):
    """One or two row tiles of sequences that are cut into pieces, between short ones, empty ones and ones without queries."""
    both = Both(gpu, B, Hk, D, 1152, 64, dtype)
    lens = [(37 * b) % 97 for b in range(B)]
    for b, n in ((1, 1100), (2, 577), (B // 2, 1152), (B - 1, 1151)):
        lens[b] = n
    both.append(1152, lens)
    q = both.rand(B, 40, H, D)
    counts = [(b * 7) % 41 for b in range(B)]
    counts[B // 2], counts[B - 1] = 40, 33
    for longest in (1152, 200000):
        both.attend(q, causal=True, longest=longest, collect=True)
        both.attend(q, counts=_i32(gpu, counts), longest=longest, collect=True)


@pytest.mark.parametrize("D,dtype,H,Hk", [(64, BF16, 3, 1), (128, F16, 4, 2), (64, F16, 2, 2)])
def test_what_prompts_give(gpu, D, dtype, H, Hk):
    """Many queries over their own tokens: most keys are seen by the later rows only."""
    both = Both(gpu, 3, Hk, D, 512, 32, dtype)
    both.append(420, [333, 420, 290])
    q = both.rand(3, 333, H, D)                              # more queries than tokens in the last
    for counts in (None, _i32(gpu, [333, 300, 1])):
        for longest in (None, 64):
            both.attend(q, causal=True, counts=counts, longest=longest, collect=True)


@pytest.mark.parametrize("n,H", [(1, 32), (8, 4), (2, 16)])
def test_attention_whose_scores_are_not_kept(gpu, n, H):
    """A capacity whose raw scores would pass 1 GiB: what is received comes from the keys again."""
    from qvggt_amd import _lib
    from qvggt_amd.kv_cache import PagedKVCache
    cap, D = (1 << 23) + 65536, 64
    need = _lib.load().qv_paged_attention_workspace(1, 1, n, H, 1, D, 70000, cap)
    assert 0 < need < 1 << 27
    cache = PagedKVCache(1, 1, D, cap, page=65536, pages=3, dtype=F16, track=True, device=gpu)
    cache.table[0, :2] = _i32(gpu, [2, 0])
    g = torch.Generator(device=gpu).manual_seed(2)
    k, v = (torch.randn(1, 70000, 1, D, generator=g, device=gpu).half() for _ in range(2))
    cache.append(k, v)
    q = torch.randn(1, n, H, D, generator=g, device=gpu).half()
    keep = np.arange(70000)[None] <= (70000 - n + np.arange(n))[:, None]
    for longest in (None, 64):                               # shares; the whole sequence
        cache.weights.zero_()
        out = cache.attention(q, causal=True, collect=True, longest=longest)
        close(out[0], q[0], k[0], v[0], keep=keep)
        received_close(cache.weights[0, :, :70000], q[0], k[0], keep=keep)
        assert not cache.weights[0, :, 70000:].any()


def test_pages_past_32_bits(gpu):
    """A pool of over 4 GiB: pages at its end, in all calls."""
    from qvggt_amd.kv_cache import PagedKVCache
    page, Hk, D, H = 1024, 8, 128, 16
    pages = (9 << 29) // (page * Hk * D * 2)                 # 4.5 GiB of keys, as much of values
    cache = PagedKVCache(2, Hk, D, 4 * page, page=page, pages=pages, dtype=BF16, track=True, device=gpu)
    small = PagedKVCache(2, Hk, D, 4 * page, page=page, dtype=BF16, track=True, device=gpu)
    cache.table.copy_(pages - 1 - torch.arange(8, device=gpu).view(2, 4))
    g = torch.Generator(device=gpu).manual_seed(2)
    k, v = (torch.randn(2, 3000, Hk, D, generator=g, device=gpu).bfloat16() for _ in range(2))
    counts = _i32(gpu, [3000, 2500])
    for n in (1, 20):
        q = torch.randn(2, n, H, D, generator=g, device=gpu).bfloat16()
        outs = []
        for c in (cache, small):
            c.append(k, v, counts=counts, start=torch.zeros_like(counts))
            c.weights.zero_()
            outs.append(c.attention(q, causal=True, collect=True))
            c.evict(1500, recent=100, first=3)
        assert torch.equal(outs[0], outs[1]) and outs[0].abs().max() > 0
        for name in ("weights", "positions", "lens", "evicted"):
            assert torch.equal(getattr(cache, name), getattr(small, name)), name
        for pool, other in ((cache.k_pages, small.k_pages), (cache.v_pages, small.v_pages)):
            assert torch.equal(pool[cache.table.long()], other[small.table.long()])
    assert not cache.k_pages[:pages - 8].any()


@pytest.mark.parametrize("n,H,Hk", [(1, 8, 2), (40, 4, 2)])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_c_entry_without_workspace(gpu, n, H, Hk, D, dtype):
    """With less workspace than it could use, or none, a call splits less; strides of a larger buffer."""
    from qvggt_amd import _lib
    from qvggt_amd import awq_inference_engine as E
    both = Both(gpu, 2, Hk, D, 6000, 64, dtype)
    both.append(6000, [6000, 777])
    c = both.cache
    wide = both.rand(2, n, H + 1, D)
    q = wide[:, :, :H]
    need = _lib.load().qv_paged_attention_workspace(0, 2, n, H, Hk, D, 6000, c.capacity)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    want = both.attend(q.contiguous(), causal=True, longest=6000)
    for given, size in ((None, 0), (ws, 16), (ws, need - 1), (ws, need)):
        out = torch.full_like(wide, 3.0)
        _lib.call("qv_paged_attention", q.data_ptr(), out.data_ptr(), 1 if dtype == BF16 else 0, c.k_pages.data_ptr(),
                  c.v_pages.data_ptr(), c.table.data_ptr(), c.lens.data_ptr(), None, 1, None, 2, n, H, Hk, D, c.page, c.slots, c.pages,
                  6000, E._i64s(*q.stride()[:3]), E._i64s(*out.stride()[:3]), D ** -0.5, None if given is None else ws.data_ptr(),
                  size, torch.cuda.current_stream().cuda_stream)
        for b in range(2):
            k, v = both.rows(b, both.ref[b].len)
            keep = np.arange(len(k))[None] <= (len(k) - n + np.arange(n))[:, None]
            close(out[b, :, :H], q[b], k, v, keep=keep)
        assert (out[:, :, H:] == 3).all()
        if size == need:
            assert torch.equal(out[:, :, :H], want)


@pytest.mark.parametrize("n,H,slots", [(1, 4, 8), (60, 2, 8), (150, 1, 200), (1, 32, 130)])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_c_entry_of_a_pool_without_pages(gpu, n, H, slots, D, dtype):
    """No page is one: queries see nothing, and nothing is received (130 slots of 65536 tokens: scores are not kept)."""
    from qvggt_amd import _lib
    from qvggt_amd import awq_inference_engine as E
    page = 65536 if slots == 130 else 64
    cap = slots * page
    q = torch.randn(2, n, H, D, device=gpu).to(dtype)
    table = torch.arange(2 * slots, dtype=torch.int32, device=gpu).view(2, slots)
    lens = _i32(gpu, [cap, 77])
    given = torch.rand(2, 1, cap, device=gpu)
    need = _lib.load().qv_paged_attention_workspace(1, 2, n, H, 1, D, cap, cap)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    for weights in (None, given.clone()):
        out = torch.full_like(q, 3.0)
        _lib.call("qv_paged_attention", q.data_ptr(), out.data_ptr(), 1 if dtype == BF16 else 0, None, None, table.data_ptr(),
                  lens.data_ptr(), None, 1, None if weights is None else weights.data_ptr(), 2, n, H, 1, D, page, slots, 0, cap,
                  E._i64s(*q.stride()[:3]), E._i64s(*out.stride()[:3]), D ** -0.5, ws.data_ptr(), need,
                  torch.cuda.current_stream().cuda_stream)
        assert not out.any()
        assert weights is None or torch.equal(weights, given)


def test_two_streams_read_one_cache(gpu):
    """Attention calls of two streams at once have workspaces of their own."""
    both = Both(gpu, 4, 2, 64, 3000, 64, F16)
    both.append(3000, [3000, 1000, 10, 2999])
    qs = [both.rand(4, 1, 8, 64) for _ in range(2)]
    want = [both.cache.attention(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, q, o in zip(streams, qs, got):
            with torch.cuda.stream(s):
                o.append(both.cache.attention(q))
    torch.cuda.synchronize()
    for o, w in zip(got, want):
        assert all(torch.equal(x, w) for x in o)


# ------------------------------------------------------------------- evict
@pytest.mark.parametrize("page,D,dtype", [(16, 64, F16), (64, 128, BF16)])
@pytest.mark.parametrize("keep,recent,first", [(100, 0, 0), (100, 30, 4), (299, 10, 0), (1, 1, 0), (1, 0, 0), (0, 0, 0), (128, 100, 28),
                                               (299, 0, 299), (300, 5, 5), (5000, 0, 0)])
def test_evict(gpu, keep, recent, first, page, D, dtype):
    both = Both(gpu, 4, 3, D, 400, page, dtype)
    both.append(300, [300, 299, 100, 7])
    for round in range(3):
        w = (torch.rand(both.cache.weights.shape, generator=both.g, device=gpu) * 8).round() / 4       # ties
        w[:, :, 10::40] = float("nan")
        w[:, :, 11::40] = float("inf")
        w[:, :, 12::40] = -1.5
        w[:, :, 13::40] = -0.0
        w[:, :, 14::40] = 0.0
        both.cache.weights.copy_(w)
        for b, r in enumerate(both.ref):
            r.weights[:] = w[b].double().cpu().numpy()
            r.evict(keep, recent, first)
        both.cache.evict(keep, recent=recent, first=first)
        both.check()
        both.append(40, [40, 0, 25, 40])
        both.check()


@pytest.mark.parametrize("tokens,keep", [(5000, 4990), (5000, 2100), (9000, 1), (70000, 50000)])
def test_evict_many(gpu, tokens, keep):
    """Over several rounds of a workgroup, even weights (all ties) and random ones."""
    both = Both(gpu, 1, 2, 64, tokens, 64, F16)
    both.append(tokens)
    w = torch.rand(both.cache.weights.shape, generator=both.g, device=gpu)
    w[:, 0] = 0.5
    both.cache.weights.copy_(w)
    both.ref[0].weights[:] = w[0].double().cpu().numpy()
    both.cache.evict(keep, recent=min(keep, 100))
    both.ref[0].evict(keep, recent=min(keep, 100))
    both.check()


# ------------------------------------------------------------ all together
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_a_stream_in_a_bounded_cache(gpu, D, dtype):
    """Packed prompts, their attention, the window that says what matters, then tokens one by one, evicted now and then."""
    from qvggt_amd import awq_inference_engine as E
    H, Hk, lens = 4, 2, (150, 3, 81)
    both = Both(gpu, 3, Hk, D, 256, 32, dtype)
    plan = E.packed_plan(lens, H, Hk, D, device=gpu)
    k, v = both.kv(sum(lens))
    q = both.rand(sum(lens), H, D)
    out = E.packed_attention(q, k, v, plan)
    both.cache.append(k, v, plan=plan)
    for r, a, n in zip(both.ref, np.cumsum((0,) + lens), lens):
        r.append(*(x[a:a + n].double().cpu().numpy() for x in (k, v)))
        close(out[a:a + n], q[a:a + n], k[a:a + n], v[a:a + n], keep=P.seen_by_frame(n, 1), matched=True)
    both.check()
    window = torch.stack([q[e - 3:e] for e in np.cumsum(lens)])
    again = both.attend(window, causal=True, collect=True)
    for b, e in enumerate(np.cumsum(lens)):
        torch.testing.assert_close(again[b].float(), out[e - 3:e].float(), rtol=0, atol=4 * {F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype] * 4)
    for i in range(20):
        both.append(1)
        both.attend(both.rand(3, 1, H, D), causal=True, collect=True)
        for b, r in enumerate(both.ref):
            r.weights[:, :r.len] = both.cache.weights[b, :, :r.len].double().cpu().numpy()
        if i % 6 == 5:
            both.cache.evict(96, recent=16, first=4)
            for r in both.ref:
                r.evict(96, recent=16, first=4)
            both.check()


def test_graph_of_a_step(gpu):
    """append, attention with collect and evict, captured once and replayed: the same bits as eagerly."""
    H, Hk, D = 4, 2, 64
    eager, graphed = (Both(gpu, 2, Hk, D, 200, 16, F16, seed=4, own=True) for _ in range(2))
    for x in (eager, graphed):
        x.append(90, [90, 40])
    k, v, q = eager.rand(2, 1, Hk, D), eager.rand(2, 1, Hk, D), eager.rand(2, 1, H, D)

    def step(c):
        c.append(k, v)
        out = c.attention(q, causal=True, collect=True)
        c.evict(92, recent=8)
        return out
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step(graphed.cache)
    for i in range(5):
        for t in (k, v, q):
            t.copy_(eager.rand(*t.shape))
        want = step(eager.cache)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for name in ("lens", "evicted", "positions", "weights"):
            assert torch.equal(getattr(graphed.cache, name), getattr(eager.cache, name)), (i, name)
        assert torch.equal(torch.nan_to_num(graphed.cache.k_pages), torch.nan_to_num(eager.cache.k_pages))
