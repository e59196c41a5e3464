"""The reference engine's attention operators over torch tensors, on libh3cuda.so.

A Python restatement of ``engine/h3-core/src/ops.rs`` of maxfridbe/sycl_minimax_h3 for this path: ``Rows`` (ops.rs
:299-324) describes token rows of ``heads x dim`` features inside a wider row-major buffer - how q, k and v sit inside
the qkv linear's output (offset i*H*D, stride 3*H*D) - and ``attention`` / ``attention_batch`` (ops.rs:405-461) check
the layouts exactly as the reference does, then call ``h3s_attention`` / ``h3s_attention_batch``.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from .native import Context, H3Error, KVCacheStruct, dt_code

_ctx: dict[tuple[int, int], Context] = {}
# the handle of a device's current stream, without a stream object for every call where torch offers that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def context(device=None) -> Context:
    """The h3s context of a device around PyTorch's current stream on it (made once per (device, stream))."""
    if device is None:
        index = torch.cuda.current_device()
    else:
        index = (device if isinstance(device, torch.device) else torch.device(device)).index or 0
    key = (index, _raw_stream(index))
    ctx = _ctx.get(key)
    if ctx is None:
        with torch.cuda.device(index):
            ctx = _ctx[key] = Context(torch.cuda.current_stream())
    return ctx


@dataclass(frozen=True)
class Rows:
    """Token rows of ``heads`` x ``dim`` features inside a wider row-major buffer: row s starts at element
    ``offset + s * stride`` of ``t`` (ops.rs:299-308)."""

    t: torch.Tensor
    offset: int
    stride: int
    tokens: int
    heads: int
    dim: int

    def layout(self):
        return (self.tokens, self.heads, self.dim, self.stride)

    def ptr(self) -> int:
        """The device address of row 0, after the reference's bounds check (ops.rs:310-323)."""
        last = self.offset + (max(self.tokens, 1) - 1) * self.stride + self.heads * self.dim
        if self.stride < self.heads * self.dim or last > self.t.numel():
            raise H3Error(f"rows of {self.heads} x {self.dim} at offset {self.offset} with stride {self.stride} do not "
                          f"fit {list(self.t.shape)}")
        if not self.t.is_contiguous():
            raise H3Error("rows must live in a contiguous tensor")
        return self.t.data_ptr() + self.offset * self.t.element_size()

    @staticmethod
    def qkv(qkv: torch.Tensor, heads: int, dim: int):
        """q, k, v as the three strided parts of a qkv linear's output [tokens, 3 * heads * dim] (dit.rs:346-350)."""
        tokens = qkv.shape[0]
        w = heads * dim
        return tuple(Rows(qkv, i * w, 3 * w, tokens, heads, dim) for i in range(3))

    @staticmethod
    def packed(x: torch.Tensor, heads: int, dim: int) -> "Rows":
        """Rows of a packed [tokens, heads * dim] tensor."""
        return Rows(x, 0, heads * dim, x.shape[0], heads, dim)


def _floats(t: torch.Tensor, what: str, n: int) -> int:
    """A float32 device tensor of exactly n values (ops.rs `floats`)."""
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise H3Error(f"{what}: {n} contiguous float32 values expected, got {list(t.shape)} {t.dtype}")
    return t.data_ptr()


def rms_rope(x: Rows, weight: torch.Tensor, eps: float, cs: torch.Tensor, rot_dim: int) -> None:
    """Per-head RMS norm (weight float32 [dim]) and the rotary rotation, in place; ``cs`` float32
    [tokens, rot_dim/2, 2] of (cos, sin) (ops.rs:326-345, kernels/h3sycl.h:165-174)."""
    ctx = context(x.t.device)
    ctx.rms_rope(x.ptr(), dt_code(x.t.dtype), x.tokens, x.heads, x.dim, x.stride,
                 _floats(weight, "the norm weight", x.dim), eps, _floats(cs, "the rotation table", x.tokens * rot_dim),
                 rot_dim)


@dataclass(frozen=True)
class Int8Linear:
    """A linear layer with int8 weights (one layer of an ``int8_convrot`` checkpoint), on the device (ops.rs:25-80):
    ``weight`` int8 [N, K], ``scale`` float32 with 1 or N values, ``bias`` float32 [N] or None, ``group`` the rotation
    group size when the weights were stored rotated."""

    weight: torch.Tensor
    scale: torch.Tensor
    bias: torch.Tensor | None = None
    group: int | None = None

    def inputs(self) -> int:
        return self.weight.shape[1]

    def outputs(self) -> int:
        return self.weight.shape[0]

    def forward(self, x: torch.Tensor, out: torch.Tensor) -> None:
        """``out = linear(x)``: x [M, K] in a float type, out [M, N] in out's type (ops.rs:45-79)."""
        n, k = self.outputs(), self.inputs()
        m = x.numel() // k
        if self.weight.dtype != torch.int8 or self.scale.dtype != torch.float32:
            raise H3Error("int8_linear: the weight must be int8 and its scale float32")
        if x.numel() != m * k or out.numel() != m * n:
            raise H3Error(f"int8_linear: x {list(x.shape)} and out {list(out.shape)} do not fit a [{n}, {k}] weight")
        ns = self.scale.numel()
        if ns != 1 and ns != n:
            raise H3Error(f"int8_linear: {ns} weight scales for {n} outputs")
        for t, what in ((x, "x"), (out, "out"), (self.weight, "the weight"), (self.scale, "the scale")):
            if not t.is_contiguous():
                raise H3Error(f"int8_linear: {what} must be contiguous")
        bias = _floats(self.bias, "the bias", n) if self.bias is not None else 0
        ctx = context(out.device)
        ctx.int8_linear(x.data_ptr(), dt_code(x.dtype), m, k, self.weight.data_ptr(), n, self.scale.data_ptr(), ns,
                        bias, out.data_ptr(), dt_code(out.dtype), self.group or 0)


def attention_causal(q: Rows, k: Rows, v: Rows, out: torch.Tensor) -> None:
    """Causal attention with grouped heads (the text encoder's call, te.rs:340-346): q has the query heads, k and v the
    key/value heads (a divisor of them), all with the same tokens and head size; out [tokens, q.heads * dim] in q's
    type (kernels/h3sycl.h:105-108)."""
    if k.layout()[1:3] != v.layout()[1:3] or k.stride != v.stride or q.tokens != k.tokens or k.tokens != v.tokens:
        raise H3Error("attention_causal: k and v must have the same layout, and q, k, v the same tokens")
    if q.dim != k.dim or k.heads == 0 or q.heads % k.heads != 0:
        raise H3Error(f"attention_causal: {q.heads} query heads over {k.heads} key/value heads of {k.dim}")
    if q.t.dtype != k.t.dtype or q.t.dtype != v.t.dtype or out.dtype != q.t.dtype:
        raise H3Error("attention_causal: q, k, v and out must have one element type")
    if out.numel() != q.tokens * q.heads * q.dim or not out.is_contiguous():
        raise H3Error(f"attention_causal: out {list(out.shape)} for {q.tokens} tokens of {q.heads} x {q.dim}")
    ctx = context(out.device)
    ctx.attention_causal(q.ptr(), k.ptr(), v.ptr(), dt_code(q.t.dtype), q.tokens, q.heads, k.heads, q.dim, q.stride,
                         k.stride, out.data_ptr())


def attention(q: Rows, k: Rows, v: Rows, out: torch.Tensor) -> None:
    """``out = softmax(q . k^T / sqrt(dim)) . v`` per head; out [tokens, heads * dim] (ops.rs:436-461)."""
    if q.layout() != k.layout() or q.layout() != v.layout():
        raise H3Error("attention: q, k and v must have the same layout")
    if out.numel() != q.tokens * q.heads * q.dim:
        raise H3Error(f"attention: out {list(out.shape)} for {q.tokens} tokens of {q.heads} x {q.dim}")
    if not out.is_contiguous():
        raise H3Error("attention: out must be contiguous")
    ctx = context(out.device)
    ctx.attention(q.ptr(), k.ptr(), v.ptr(), dt_code(q.t.dtype), q.tokens, q.heads, q.dim, q.stride, out.data_ptr(),
                  dt_code(out.dtype))


def attention_batch(q: Rows, k: Rows, v: Rows, seqs: int, out: torch.Tensor) -> None:
    """Attention over ``seqs`` independent sequences of ``q.tokens / seqs`` tokens each, in one call (ops.rs:405-434)."""
    if q.layout() != k.layout() or q.layout() != v.layout():
        raise H3Error("attention_batch: q, k and v must have the same layout")
    if seqs == 0 or q.tokens % seqs != 0:
        raise H3Error(f"attention_batch: {q.tokens} tokens are not {seqs} equal sequences")
    if out.numel() != q.tokens * q.heads * q.dim:
        raise H3Error(f"attention_batch: out {list(out.shape)} for {q.tokens} tokens of {q.heads} x {q.dim}")
    ctx = context(out.device)
    ctx.attention_batch(q.ptr(), k.ptr(), v.ptr(), dt_code(q.t.dtype), seqs, q.tokens // seqs, q.heads, q.dim, q.stride,
                        out.data_ptr(), dt_code(out.dtype))


def attention_rms_rope(q: Rows, k: Rows, v: Rows, out: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
                       eps: float, cs: torch.Tensor, rot_dim: int) -> None:
    """A denoiser block's ``rms_rope(q)``, ``rms_rope(k)``, ``attention(q, k, v, out)`` in one call (dit.rs:347-350):
    q and k are left normalised and rotated in place, as the two ``rms_rope`` calls leave them."""
    if q.layout() != k.layout() or q.layout() != v.layout():
        raise H3Error("attention_rms_rope: q, k and v must have the same layout")
    if out.numel() != q.tokens * q.heads * q.dim or not out.is_contiguous():
        raise H3Error(f"attention_rms_rope: out {list(out.shape)} for {q.tokens} tokens of {q.heads} x {q.dim}")
    ctx = context(out.device)
    ctx.attention_rms_rope(q.ptr(), k.ptr(), v.ptr(), dt_code(q.t.dtype), q.tokens, q.heads, q.dim, q.stride,
                           out.data_ptr(), dt_code(out.dtype), _floats(q_norm, "the q norm weight", q.dim),
                           _floats(k_norm, "the k norm weight", q.dim), eps,
                           _floats(cs, "the rotation table", q.tokens * rot_dim), rot_dim)


# ---- the text model token by token: an 8-bit key/value cache and 4-bit linear layers (include/h3cuda.h) ----

PAGE = 64  # tokens of a page


def _part(t: torch.Tensor, what: str, dtype: torch.dtype, shape, device) -> int:
    """The address of a contiguous tensor of this type, shape and device."""
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.device != device:
        raise H3Error(f"{what}: contiguous {dtype} {list(shape)} on {device} expected, got {t.dtype} {list(t.shape)} on "
                      f"{t.device}")
    return t.data_ptr()


def _on_gpu(device: torch.device, what: str) -> None:
    if device.type != "cuda":
        raise H3Error(f"{what}: the tensors must be on a GPU, not on {device}")


@dataclass(frozen=True, eq=False)
class KVCache:
    """The keys and values of a batch of growing sequences in 8 bits (``h3s_kv_cache``): ``k``, ``v`` int8 [pages, heads,
    64, dim] with ``k_scale``, ``v_scale`` float32 [pages, heads]; ``tail_k``, ``tail_v`` [seqs, heads, 64, dim] in the
    rows' type, the tokens that do not fill a page yet; ``table`` int32 [seqs, width] page ids, ``lens`` int32 [seqs] tokens
    (those of the current call included); ``weight`` float32 [pages, heads, 64] and ``tail_weight`` [seqs, heads, 64], the
    attention weight that each token has received, where tokens are evicted by it. dim is 64 or 128.

    ``lens`` and ``table`` are the caller's to change, on the device, between calls; which pages are free is the caller's
    to keep. The tensors themselves stay: their addresses are taken down once."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    tail_k: torch.Tensor
    tail_v: torch.Tensor
    table: torch.Tensor
    lens: torch.Tensor
    weight: torch.Tensor | None = None
    tail_weight: torch.Tensor | None = None

    def __post_init__(self):
        if self.k.dim() != 4 or self.k.shape[2] != PAGE or self.table.dim() != 2:
            raise H3Error(f"KVCache: k [pages, heads, {PAGE}, dim] and table [seqs, width] expected, got {list(self.k.shape)} "
                          f"and {list(self.table.shape)}")
        pages, heads, _, dim = self.k.shape
        seqs, width = self.table.shape
        dt, dev, i8, f32, i32 = self.tail_k.dtype, self.k.device, torch.int8, torch.float32, torch.int32
        if dim not in (64, 128):
            raise H3Error(f"KVCache: heads of 64 or 128 features (got {dim})")
        if (self.weight is None) != (self.tail_weight is None):
            raise H3Error("KVCache: weight and tail_weight come together")
        s = KVCacheStruct(
            _part(self.k, "KVCache: k", i8, self.k.shape, dev), _part(self.v, "KVCache: v", i8, self.k.shape, dev),
            _part(self.k_scale, "KVCache: k_scale", f32, (pages, heads), dev),
            _part(self.v_scale, "KVCache: v_scale", f32, (pages, heads), dev),
            _part(self.tail_k, "KVCache: tail_k", dt, (seqs, heads, PAGE, dim), dev),
            _part(self.tail_v, "KVCache: tail_v", dt, (seqs, heads, PAGE, dim), dev),
            None if self.weight is None else _part(self.weight, "KVCache: weight", f32, (pages, heads, PAGE), dev),
            None if self.tail_weight is None else _part(self.tail_weight, "KVCache: tail_weight", f32, (seqs, heads, PAGE), dev),
            _part(self.table, "KVCache: table", i32, (seqs, width), dev), _part(self.lens, "KVCache: lens", i32, (seqs,), dev),
            pages, seqs, width, heads, dim, dt_code(dt))
        object.__setattr__(self, "_sizes", (pages, heads, dim, seqs, width))
        object.__setattr__(self, "_device", dev)
        object.__setattr__(self, "_struct", s)
        object.__setattr__(self, "_ptr", ctypes.addressof(s))
        object.__setattr__(self, "_work", {})

    @staticmethod
    def empty(pages: int, seqs: int, width: int, heads: int, dim: int, dtype: torch.dtype, device="cuda",
              weights: bool = False) -> "KVCache":
        """A cache without a token: room for ``pages`` pages, ``width`` of them at most for each of ``seqs`` sequences. The
        table is -1 throughout: pages are given out by writing their ids into it."""
        f32, kw = torch.float32, {"device": device}
        return KVCache(torch.zeros(pages, heads, PAGE, dim, dtype=torch.int8, **kw),
                       torch.zeros(pages, heads, PAGE, dim, dtype=torch.int8, **kw),
                       torch.zeros(pages, heads, dtype=f32, **kw), torch.zeros(pages, heads, dtype=f32, **kw),
                       torch.zeros(seqs, heads, PAGE, dim, dtype=dtype, **kw),
                       torch.zeros(seqs, heads, PAGE, dim, dtype=dtype, **kw),
                       torch.full((seqs, width), -1, dtype=torch.int32, **kw), torch.zeros(seqs, dtype=torch.int32, **kw),
                       torch.zeros(pages, heads, PAGE, dtype=f32, **kw) if weights else None,
                       torch.zeros(seqs, heads, PAGE, dtype=f32, **kw) if weights else None)

    def _rows(self, what: str, x: Rows) -> int:
        if x.dim != self._sizes[2] or x.t.dtype != self.tail_k.dtype or x.t.device != self._device:
            raise H3Error(f"{what}: {x.t.dtype} rows with heads of {x.dim} on {x.t.device}, but the cache has {self.tail_k.dtype} "
                          f"and {self.k.shape[3]} on {self.k.device}")
        return x.ptr()

    def _starts(self, what: str, starts: torch.Tensor) -> int:
        return _part(starts, what, torch.int32, (self._sizes[3] + 1,), self._device)


def kv_append(cache: KVCache, k: Rows, v: Rows, starts: torch.Tensor, max_new: int | None = None) -> None:
    """The rows of new tokens into the cache (``h3s_kv_append``): sequence b's are the rows starts[b] .. starts[b+1] - 1 of
    k and v, and the last ones of its ``cache.lens[b]`` tokens. A block of 64 tokens that is full is quantised, the others
    stay in the tail as they are. ``max_new`` (about the most that one sequence gets) only divides the work."""
    if k.layout() != v.layout():
        raise H3Error("kv_append: k and v must have the same layout")
    if k.heads != cache._sizes[1]:
        raise H3Error(f"kv_append: {k.heads} heads for a cache of {cache._sizes[1]}")
    kp, vp, sp = cache._rows("kv_append", k), cache._rows("kv_append", v), cache._starts("kv_append: starts", starts)
    _on_gpu(cache._device, "kv_append")
    context(cache._device).kv_append(cache._ptr, kp, vp, k.tokens, k.stride, sp, max_new or 0)


def attention_cached(q: Rows, cache: KVCache, starts: torch.Tensor, out: torch.Tensor, max_new: int | None = None,
                     max_len: int | None = None, accumulate: bool = False) -> None:
    """Causal attention with grouped heads over the cache (``h3s_attention_cached``): query rows starts[b] .. starts[b+1] - 1
    are the last tokens of sequence b and see every token up to their own; out [q.tokens, q.heads * dim]. A row that sees
    nothing is 0; rows behind the last sequence are left as they were. ``accumulate`` adds the weight that every token
    receives to ``cache.weight`` (a second pass over the keys, made for single tokens: dear for a long prompt). Sums are held
    in float32; the softmax's weights enter the products as fp16, or two fp16 terms for float32 rows. ``max_new`` and
    ``max_len`` (about the most new tokens, and the longest sequence) only divide the work."""
    heads, dim = cache._sizes[1:3]
    if q.heads == 0 or q.heads % heads != 0:
        raise H3Error(f"attention_cached: {q.heads} query heads over {heads} key/value heads")
    if accumulate and cache.weight is None:
        raise H3Error("attention_cached: the cache keeps no weights")
    if out.dtype != q.t.dtype or out.numel() != q.tokens * q.heads * dim or not out.is_contiguous() or out.device != q.t.device:
        raise H3Error(f"attention_cached: out {list(out.shape)} {out.dtype} for {q.tokens} tokens of {q.heads} x {dim} in "
                      f"{q.t.dtype}")
    qp, sp = cache._rows("attention_cached", q), cache._starts("attention_cached: starts", starts)
    _on_gpu(cache._device, "attention_cached")
    ctx = context(cache._device)
    key = (q.tokens, q.heads, max_new, max_len, accumulate)
    nbytes = cache._work.get(key)
    if nbytes is None:
        if len(cache._work) >= 256:
            cache._work.clear()
        nbytes = cache._work[key] = ctx.attention_cached_work(cache._ptr, q.tokens, q.heads, max_new or 0, max_len or 0, accumulate)
    work = torch.empty(nbytes, dtype=torch.uint8, device=cache._device) if nbytes else None
    ctx.attention_cached(cache._ptr, qp, q.tokens, q.heads, q.stride, sp, max_new or 0, max_len or 0, out.data_ptr(),
                         int(accumulate), work.data_ptr() if nbytes else 0, nbytes)


def kv_evict(cache: KVCache, spare: torch.Tensor, budget: int, sinks: int = 4, recent: int = PAGE) -> None:
    """Cuts every sequence longer than ``budget`` tokens (a multiple of 64) to it (``h3s_kv_evict``): each head keeps its
    first ``sinks`` and last ``recent`` tokens and those of the others with the largest ``cache.weight``. They move to the
    pages ``spare`` int32 [seqs, budget / 64], which change places with the sequence's old ones in ``cache.table``."""
    if cache.weight is None:
        raise H3Error("kv_evict: the cache keeps no weights")
    if budget <= 0 or budget % PAGE:
        raise H3Error(f"kv_evict: the budget must be a multiple of {PAGE} (got {budget})")
    if sinks < 0 or recent < 0 or sinks + recent > budget:
        raise H3Error(f"kv_evict: {sinks} first and {recent} last tokens do not fit a budget of {budget}")
    seqs, heads = cache.table.shape[0], cache.k.shape[1]
    sp = _part(spare, "kv_evict: spare", torch.int32, (seqs, budget // PAGE), cache.k.device)
    _on_gpu(cache.k.device, "kv_evict")
    nbytes = 4 * seqs * heads * budget
    work = torch.empty(nbytes, dtype=torch.uint8, device=cache.k.device)
    context(cache.k.device).kv_evict(cache._ptr, sp, budget, sinks, recent, work.data_ptr(), nbytes)


@dataclass(frozen=True, eq=False)
class Int4Linear:
    """A linear layer with 4-bit weights W[n, k] = scale[k // group, n] * (code[n, k] - zero[k // group, n]) for a few rows
    at a time (``h3s_int4_linear``): ``tiles`` the codes as ``pack`` lays them out, ``scale`` (and ``zero``, or None: 8)
    [ceil(inputs / group), outputs] in a float type, ``group`` 32, 64, 128 or 0 (one scale per output), ``bias`` float32
    [outputs] or None."""

    tiles: torch.Tensor
    scale: torch.Tensor
    n: int
    k: int
    group: int
    zero: torch.Tensor | None = None
    bias: torch.Tensor | None = None

    def __post_init__(self):
        if self.group not in (0, 32, 64, 128):
            raise H3Error(f"int4_linear: groups of 32, 64 or 128 inputs, or 0 (got {self.group})")
        dev, groups = self.tiles.device, -(-self.k // self.group) if self.group else 1
        _part(self.tiles, "int4_linear: tiles", torch.int32, (-(-self.n // 16), -(-self.k // 64), 128), dev)
        dt_code(self.scale.dtype)
        _part(self.scale, "int4_linear: scale", self.scale.dtype, (groups, self.n), dev)
        if self.zero is not None:
            _part(self.zero, "int4_linear: zero", self.scale.dtype, (groups, self.n), dev)
        if self.bias is not None:
            _part(self.bias, "int4_linear: bias", torch.float32, (self.n,), dev)

    @staticmethod
    def pack(codes: torch.Tensor, scale: torch.Tensor, group: int, zero: torch.Tensor | None = None,
             bias: torch.Tensor | None = None) -> "Int4Linear":
        """From codes uint8 [outputs, inputs / 2], input 2 i in the low four bits of byte i (``h3s_int4_pack``)."""
        if codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.is_contiguous():
            raise H3Error(f"int4_linear: contiguous uint8 codes [outputs, inputs / 2] expected, got {list(codes.shape)} {codes.dtype}")
        _on_gpu(codes.device, "int4_linear")
        n, k = codes.shape[0], codes.shape[1] * 2
        tiles = torch.empty(-(-n // 16), -(-k // 64), 128, dtype=torch.int32, device=codes.device)
        context(codes.device).int4_pack(codes.data_ptr(), n, k, tiles.data_ptr())
        return Int4Linear(tiles, scale, n, k, group, zero, bias)

    def inputs(self) -> int:
        return self.k

    def outputs(self) -> int:
        return self.n

    def forward(self, x: torch.Tensor, out: torch.Tensor) -> None:
        """``out = linear(x)``: x [M, inputs] in a float type, out [M, outputs] in out's type. Infinities and NaN come out as the
        formula has them, also where the float32 sums do not hold them."""
        m = x.numel() // self.k if self.k else 0
        if x.numel() != m * self.k or out.numel() != m * self.n:
            raise H3Error(f"int4_linear: x {list(x.shape)} and out {list(out.shape)} do not fit a [{self.n}, {self.k}] weight")
        for t, what in ((x, "x"), (out, "out")):
            if not t.is_contiguous() or t.device != self.tiles.device:
                raise H3Error(f"int4_linear: {what} must be contiguous, on {self.tiles.device}")
        x_dt, out_dt = dt_code(x.dtype), dt_code(out.dtype)
        _on_gpu(self.tiles.device, "int4_linear")
        context(self.tiles.device).int4_linear(
            x.data_ptr(), x_dt, m, self.k, self.tiles.data_ptr(), self.n, self.scale.data_ptr(),
            self.zero.data_ptr() if self.zero is not None else 0, dt_code(self.scale.dtype), self.group,
            self.bias.data_ptr() if self.bias is not None else 0, out.data_ptr(), out_dt)
