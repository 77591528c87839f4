"""Keys and values of earlier tokens in 8 bits, and the attention that reads them.

The streaming side of the attention ops: a program that sees frames (or tokens)
one after another rotates the new queries and keys (``rope_axes``), appends
the new keys and values here and lets the new queries attend to all of them.
No reference counterpart (VGGT's own global attention sees all frames at once;
the reference extension's decode attention keeps a 16-bit cache of its own layout).
"""
from __future__ import annotations

import torch

from . import _lib
from .awq_inference_engine import (_device, _dtype_code, _fail, _kv_query, _kv_rows, _kv_strides, _kv_workspace_bytes,
                                   _on_gpu, _ptr, _stream)

BLOCK = 64   # tokens of a block
MOST_BLOCKS = (1 << 23) - 1   # of a sequence, as the C entries count them


class Int8KVCache:
    """Int8 keys and values of ``batch`` sequences of up to ``capacity`` tokens
    (rounded up to whole blocks of 64), ``kv_heads`` heads of 64 or 128 dims.

    Each block of 64 tokens has one scale for each head: the smallest number
    of four significant bits that is at least amax / 127 (so that a cached value,
    code * scale, has the 11 bits of an fp16 number, and attention uses it without a
    further rounding).  A NaN or infinity makes all of its (block, head) NaN, and what
    attends to a token of it, until the block is begun again.  A block that is
    filled by several calls keeps the largest scale that it needed, and its
    earlier codes are rounded again when that grows.

    ``lens`` (int32, on the GPU) holds the tokens of each sequence.  ``append``,
    ``values``, ``attention`` and ``reset`` only enqueue work, in stream order, and can
    be captured into graphs: a replayed ``append`` goes on from the ``lens`` that it
    finds.  ``load_codes`` and ``save_codes`` wait for the GPU.  One cache is written
    by one stream at a time.
    """

    def __init__(self, batch: int, kv_heads: int, head_dim: int, capacity: int, device="cuda"):
        what = "Int8KVCache"
        if head_dim not in (64, 128):
            _fail(f"{what}: head_dim must be 64 or 128, got {head_dim}")
        if not (1 <= batch <= 32767 and 1 <= kv_heads <= 65535 and 1 <= capacity <= MOST_BLOCKS * BLOCK):
            _fail(f"{what}: bad batch {batch}, kv_heads {kv_heads} or capacity {capacity}")
        self.batch, self.kv_heads, self.head_dim = batch, kv_heads, head_dim
        self.blocks = -(-capacity // BLOCK)
        self.capacity = self.blocks * BLOCK
        kw = dict(device=torch.device(device))
        shape = (batch, kv_heads, self.blocks, BLOCK * head_dim)
        self.k_codes = torch.zeros(shape, dtype=torch.int8, **kw)
        self.v_codes = torch.zeros(shape, dtype=torch.int8, **kw)
        self.k_scales = torch.zeros(shape[:3], dtype=torch.float32, **kw)
        self.v_scales = torch.zeros(shape[:3], dtype=torch.float32, **kw)
        self.lens = torch.zeros(batch, dtype=torch.int32, **kw)
        self._tickets = torch.zeros(batch * (kv_heads + 1) * _lib.QV_KV8_TICKETS, dtype=torch.int32, **kw)
        self._bound = 0

    # ------------------------------------------------------------- contents
    def reset(self) -> None:
        """Forget all tokens (``lens`` becomes 0; the blocks are written anew as they fill)."""
        self.lens.zero_()
        self._bound = 0

    def _per_sequence(self, t: torch.Tensor | None, what: str, name: str) -> None:
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (self.batch,) or not t.is_contiguous()):
            _fail(f"{what}: {name} must be contiguous int32 ({self.batch},), got {t.dtype} {tuple(t.shape)}")

    def append(self, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None,
               start: torch.Tensor | None = None) -> None:
        """Append k, v (B, n, kv_heads, head_dim), fp16 or bf16, and advance ``lens``.

        counts (B,) int32: how many of the n tokens each sequence has (the rest is
        padding; not read).  start (B,) int32: append behind that many tokens in
        place of ``lens``; what the sequence held behind them is dropped.  Where start
        passes ``lens`` the tokens in between are what the blocks hold there: zeros in a
        new cache, or what was dropped or forgotten.  Tokens past the capacity are
        dropped (``lens`` stops there)."""
        what = "Int8KVCache.append"
        dt = _dtype_code(k, what)
        want = (self.batch, self.kv_heads, self.head_dim)
        for name, t in (("k", k), ("v", v)):
            if t.dim() != 4 or (t.shape[0], *t.shape[2:]) != want or t.shape[1] != k.shape[1] or t.dtype != k.dtype:
                _fail(f"{what}: {name} must be {k.dtype} ({want[0]}, n, {want[1]}, {want[2]}), "
                      f"got {t.dtype} {tuple(t.shape)}")
        n = k.shape[1]
        if n > self.capacity:
            _fail(f"{what}: {n} tokens do not fit a cache of {self.capacity}")
        self._per_sequence(counts, what, "counts")
        self._per_sequence(start, what, "start")
        dev = _on_gpu(k, v, counts, start, self.lens, what=what)
        k, v = _kv_rows(k), _kv_rows(v)
        with _device(dev):
            _lib.call("qv_kv8_append", _ptr(k), _ptr(v), dt, _ptr(self.k_codes), _ptr(self.v_codes), _ptr(self.k_scales),
                      _ptr(self.v_scales), _ptr(self.lens if start is None else start), _ptr(self.lens),
                      _ptr(self._tickets), _ptr(counts), self.batch, n, self.kv_heads, self.head_dim, self.blocks,
                      _kv_strides(k), _kv_strides(v), _stream(dev))
        # how long a sequence may be by now: a hint for the attention's split of the keys.  Behind a
        # start, which lies on the GPU, a sequence may have any length.
        own = start is None or start.data_ptr() == self.lens.data_ptr()
        self._bound = min(self.capacity, self._bound + n) if own else self.capacity

    def values(self, n: int | None = None, first: torch.Tensor | None = None, dtype: torch.dtype = torch.float32):
        """The cached (keys, values) of n tokens (default: the capacity) of each sequence
        from token first[b] (int32 (B,); default 0) on, (B, n, kv_heads, head_dim);
        zero behind ``lens``.  float32 holds them exactly, float16 those of blocks whose
        largest lies between 2^-14 and 2^15 (a value may come back half a step larger)."""
        what = "Int8KVCache.values"
        n = self.capacity if n is None else n
        if not 0 <= n < 1 << 29:
            _fail(f"{what}: bad number of tokens {n}")
        if dtype not in (torch.float32, torch.float16, torch.bfloat16):
            _fail(f"{what}: dtype must be float32, float16 or bfloat16, got {dtype}")
        self._per_sequence(first, what, "first")
        dev = _on_gpu(self.lens, first, what=what)
        shape = (self.batch, n, self.kv_heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=self.lens.device) for _ in range(2))
        dt = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}[dtype]
        with _device(dev):
            _lib.call("qv_kv8_values", _ptr(self.k_codes), _ptr(self.v_codes), _ptr(self.k_scales), _ptr(self.v_scales),
                      _ptr(self.lens), _ptr(first), _ptr(k), _ptr(v), dt, self.batch, n, self.kv_heads, self.head_dim,
                      self.blocks, _stream(dev))
        return k, v

    # ------------------------------------------------------------ attention
    def attention(self, q: torch.Tensor, scale: float | None = None, causal: bool = False,
                  counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  longest: int | None = None) -> torch.Tensor:
        """Attention of q (B, n, heads, head_dim), fp16 or bf16, over the cached tokens of
        each sequence; heads a multiple of kv_heads, scale head_dim**-0.5 by default.

        causal: the queries are the sequence's last n tokens, each sees the tokens
        up to its own.  counts int32 (B,): how many of the n queries each sequence
        has; the rows of ``out`` behind them are left as they were (zero in a new
        out).  A query that sees no token gives zeros.  ``out`` must not overlap q.
        longest: about how many tokens the longest sequence has, for the split of the
        keys over the chip, and for nothing else: any number gives the result.  By
        default the tokens of the calls to ``append`` so far (those of a graph's capture,
        not of its replays), the capacity once one had a ``start``: a program that goes
        back and forth in a large cache, or replays, does well to say it.
        Of the values that a query sees, what lies below 2^-60 of the largest block scale
        among them may be lost, whatever their weights (only bfloat16 ones span so far).
        Returns (B, n, heads, head_dim)."""
        what = "Int8KVCache.attention"
        dt, scale = _kv_query(q, self.kv_heads, out, scale, what)
        B, n, H, D = q.shape
        if B != self.batch or D != self.head_dim:
            _fail(f"{what}: q must be ({self.batch}, n, heads, {self.head_dim}), got {tuple(q.shape)}")
        self._per_sequence(counts, what, "counts")
        if longest is not None and longest < 0:
            _fail(f"{what}: longest must not be negative, got {longest}")
        keys = self._bound if longest is None else min(self.capacity, int(longest))
        dev = _on_gpu(q, counts, out, self.lens, what=what)
        q = _kv_rows(q)
        if out is None:
            new = torch.empty if counts is None else torch.zeros
            out = new((B, n, H, D), dtype=q.dtype, device=q.device)
        ws_bytes = _kv_workspace_bytes(1, B, n, H, self.kv_heads, D, keys)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
        with _device(dev):
            _lib.call("qv_kv8_attention", _ptr(q), _ptr(out), dt, _ptr(self.k_codes), _ptr(self.v_codes), _ptr(self.k_scales),
                      _ptr(self.v_scales), _ptr(self.lens), _ptr(counts), 1 if causal else 0, B, n, H, self.kv_heads, D,
                      self.blocks, keys, _kv_strides(q), _kv_strides(out), scale, _ptr(ws), ws_bytes, _stream(dev))
        return out

    # ----------------------------------------------- codes in token order
    def _order(self):
        """Where dim d of token t lies in a block: (64, head_dim) offsets of the keys' and the values' codes."""
        t = torch.arange(BLOCK)[:, None]
        d = torch.arange(self.head_dim)[None]
        key = ((t // 32 * (self.head_dim // 32) + d // 32) * 64 + d // 16 % 2 * 32 + t % 32) * 16 + d % 16
        group, at = t // 16, t % 16
        val = ((d // 32 * 2 + group // 2) * 64 + at // 4 % 2 * 32 + d % 32) * 16 + group % 2 * 8 + at // 8 * 4 + at % 4
        return key.to(self.lens.device), val.to(self.lens.device)

    def load_codes(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                   lens: torch.Tensor) -> None:
        """Fill the cache from codes in token order, int8 (B, tokens, kv_heads, head_dim),
        tokens a multiple of 64 up to the capacity, and float32 scales (B, tokens / 64,
        kv_heads) of at most four significant bits: a cache that was saved with ``save_codes``."""
        what = "Int8KVCache.load_codes"
        B, H, D = self.batch, self.kv_heads, self.head_dim
        nb = k_codes.shape[1] // BLOCK if k_codes.dim() == 4 else 0
        for name, c, s in (("k", k_codes, k_scales), ("v", v_codes, v_scales)):
            if c.dtype != torch.int8 or tuple(c.shape) != (B, nb * BLOCK, H, D) or nb > self.blocks:
                _fail(f"{what}: {name}_codes must be int8 ({B}, tokens, {H}, {D}), tokens a multiple of {BLOCK} up to "
                      f"{self.capacity}, got {c.dtype} {tuple(c.shape)}")
            if s.dtype != torch.float32 or tuple(s.shape) != (B, nb, H):
                _fail(f"{what}: {name}_scales must be float32 ({B}, {nb}, {H}), got {s.dtype} {tuple(s.shape)}")
            m = torch.frexp(s)[0] * 16
            if not bool(((s == 0) | s.isnan() | ((m == m.round()) & (s >= 2.0 ** -120) & ~s.isinf())).all()):
                _fail(f"{what}: {name}_scales must be 0 or positive numbers of four significant bits")
            if bool((c == -128).any()):
                _fail(f"{what}: {name}_codes must lie in -127..127")
        if lens.dtype != torch.int32 or tuple(lens.shape) != (B,) or not bool(((lens >= 0) & (lens <= nb * BLOCK)).all()):
            _fail(f"{what}: lens must be int32 ({B},), 0 to {nb * BLOCK}")
        _on_gpu(k_codes, k_scales, v_codes, v_scales, lens, self.lens, what=what)
        for order, c, s, codes, scales in zip(self._order(), (k_codes, v_codes), (k_scales, v_scales),
                                              (self.k_codes, self.v_codes), (self.k_scales, self.v_scales)):
            blocks = c.view(B, nb, BLOCK, H, D) if c.is_contiguous() else c.reshape(B, nb, BLOCK, H, D)
            back = torch.empty(BLOCK * D, dtype=torch.long, device=c.device)
            back[order.reshape(-1)] = torch.arange(BLOCK * D, device=c.device)
            codes[:, :, :nb] = blocks.permute(0, 3, 1, 2, 4).reshape(B, H, nb, BLOCK * D)[..., back]
            scales[:, :, :nb] = s.transpose(1, 2)
        self.lens.copy_(lens)
        self._bound = nb * BLOCK

    def save_codes(self):
        """(k_codes, k_scales, v_codes, v_scales, lens) as ``load_codes`` takes them; copies."""
        B, H, D, nb = self.batch, self.kv_heads, self.head_dim, self.blocks
        out = []
        for order, codes, scales in zip(self._order(), (self.k_codes, self.v_codes), (self.k_scales, self.v_scales)):
            c = codes[..., order.reshape(-1)].view(B, H, nb, BLOCK, D).permute(0, 2, 3, 1, 4)
            out += [c.reshape(B, nb * BLOCK, H, D), scales.transpose(1, 2).contiguous()]
        return (*out, self.lens.clone())
