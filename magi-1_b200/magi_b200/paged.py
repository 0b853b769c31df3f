"""Token-paged 8-bit cache, attention over it, and rotary embedding by position.

ChunkPagedKVCache (ops.py) keeps whole chunks of video tokens and books them on the host; here a page holds a few tokens of
a sequence and the books are device tensors, so that appending one token to every sequence of a batch - or forking, copying,
freeing and compacting sequences - needs no host synchronisation and can be captured in a CUDA graph.  A step of a serving
loop: rotary(q), rotary(k) -> reserve -> append -> paged_attn.
"""
import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import PagedAttnParams, RotaryParams, TokenCache, check, lib
from .ops import HEAD_DIM, KERNEL_LAUNCHES, Context

MAX_ENTRIES = 1024
_INT32_MAX = 2 ** 31 - 1
_ATTN_BYTES, _ROTARY_BYTES = C.sizeof(PagedAttnParams), C.sizeof(RotaryParams)


def _on(stream, device):
    """Raw handle of the stream the call runs on: the device's current one unless one is given."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device.index)
    if stream.device != device:
        raise ValueError(f"stream belongs to {stream.device}, the tensors to {device}")
    return stream.cuda_stream


def _empty_on(stream, shape, dtype, device):
    """torch.empty whose memory belongs to `stream` (the caching allocator hands it on in that stream's order)."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _index(t, name: str, device, n: Optional[int] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor on {device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, got {t.shape[0]}")
    return t


def _fit(t, name: str) -> None:
    """The library counts in 32 bits."""
    rows, heads, _ = t.shape
    if rows > _INT32_MAX or heads > _INT32_MAX:
        raise ValueError(f"{name} is beyond 32-bit sizes")


def _rows(t, name: str, device, heads: Optional[int] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.bfloat16 or t.dim() != 3 or t.shape[2] != HEAD_DIM \
            or t.stride(2) != 1 or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be a bf16 [tokens, {heads if heads is not None else 'heads'}, {HEAD_DIM}] tensor on {device} "
                         "with a contiguous last dim")
    _fit(t, name)
    return t


def _layer(layer, cache) -> int:
    return min(max(int(layer), -1), cache.n_layers)  # the library refuses both ends; nothing wraps on its way there


def _one_place_each(t: torch.Tensor, name: str) -> None:
    """Refuse a result tensor in which two elements share memory (a broadcast view)."""
    if t.is_contiguous():
        return
    span = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: d[1]):
        if size > 1:
            if stride < span:
                raise ValueError(f"{name} must not hold two elements in one place")
            span = stride * (size - 1) + span


def _same_view(a: torch.Tensor, b: torch.Tensor) -> bool:
    """b's elements are a's (b may have more rows): the strides count where there is more than one element."""
    return a.data_ptr() == b.data_ptr() and all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _reach(t: torch.Tensor) -> int:
    """Elements from a view's first to its last, both counted."""
    return 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views of one type may share memory, b one without an element twice.  Exact where their strides are the same (two
    groups of heads of a packed tensor lie between each other); views that reach into each other with other strides count as
    sharing."""
    if not a.numel() or not b.numel():
        return False
    size = a.element_size()
    gap = b.data_ptr() - a.data_ptr()
    if gap >= _reach(a) * size or -gap >= _reach(b) * size:
        return False
    dims = [(n, m, s, t) for n, m, s, t in zip(a.shape, b.shape, a.stride(), b.stride()) if n > 1 or m > 1]
    if gap % size or any(s != t and n > 1 and m > 1 for n, m, s, t in dims):
        return True
    # a's index minus b's, per dim, has to make up the gap: from the widest stride down, what the narrower ones cannot reach rules out
    dims = sorted(((s if n > 1 else t, n, m) for n, m, s, t in dims), reverse=True)

    def meets(gap, k):
        if k == len(dims):
            return gap == 0
        stride, n, m = dims[k]
        up = sum(s * (x - 1) for s, x, _ in dims[k + 1:])
        down = sum(s * (y - 1) for s, _, y in dims[k + 1:])
        if stride == 0:
            return meets(gap, k + 1)
        lo, hi = max(-((up - gap) // stride), 1 - m), min((gap + down) // stride, n - 1)
        return any(meets(gap - d * stride, k + 1) for d in range(lo, hi + 1))

    return meets(gap // size, 0)


def _itself_or_apart(x: torch.Tensor, out: torch.Tensor, name: str) -> None:
    """Refuse an `out` that shares memory with x in another way than being x.  The usual cases come first and cost little."""
    gap = out.data_ptr() - x.data_ptr()
    if gap == 0 and x.stride() == out.stride():
        return
    first = x if gap > 0 else out
    (n, h, d), (t, s, _) = first.shape, first.stride()
    if abs(gap) >= ((n - 1) * t + (h - 1) * s + d) * x.element_size() or _same_view(x, out) or not _overlap(x, out):
        return
    raise ValueError(f"out may be {name} itself, or memory apart from it, not another view of the same")


class TokenPagedKVCache:
    """Pages of page_tokens tokens, e4m3 codes with a power-of-two scale per (page, kv head), K and V separate.

    Device state, all of it plain tensors that may be read at any time (and saved and put back with copy_, all three books
    together, to rewind all sequences at once; a page keeps the scale that it had grown to.  A length alone is not to be changed:
    the pages behind it would stay taken):
      k8, v8 [n_layers, n_pages, n_kv_heads, page_tokens, 128] float8_e4m3fn; k_scale, v_scale [n_layers, n_pages, n_kv_heads]
      page_table [max_seqs, max_pages_per_seq] int32 (-1 = none); seq_lens [max_seqs] int32; page_refs [n_pages] int32
      page_uses [n_pages] int32, scale_uses [2, n_layers, n_pages, n_kv_heads] int32: the uses that reserve made of a page, and the one its
      scale was set in (whoever puts codes and scales back puts these back with them)
    A page id names the same page in every layer.  The index arguments of the methods are int32 tensors on the cache's
    device, at most 1024 entries, no sequence twice (attention excepted); they and the books stay as they are while a call
    that reads them runs.  A book-keeping call that cannot be served - an index out of range, a sequence named twice or longer
    than its table row, too few free pages - changes nothing and shows in Context.status(): E_RANGE or E_NOMEM.  Calls on one
    cache must be stream-ordered, except that append and paged_attn of different layers may overlap."""

    def __init__(self, n_layers: int, n_pages: int, page_tokens: int, n_kv_heads: int, max_seqs: int, max_pages_per_seq: int,
                 device=None):
        sizes = dict(n_layers=n_layers, n_pages=n_pages, page_tokens=page_tokens, n_kv_heads=n_kv_heads, max_seqs=max_seqs,
                     max_pages_per_seq=max_pages_per_seq)
        for name, v in sizes.items():
            if int(v) <= 0:
                raise ValueError(f"{name} must be positive, got {v}")
            setattr(self, name, int(v))
        if self.page_tokens not in (16, 32, 64, 128):
            raise ValueError(f"page_tokens must be 16, 32, 64 or 128, got {page_tokens}")
        self.ctx = Context.get(device)
        dev = self.device = torch.device("cuda", self.ctx.device)
        shape = (self.n_layers, self.n_pages, self.n_kv_heads, self.page_tokens, HEAD_DIM)
        # zero-filled once: attention multiplies what lies behind a sequence's end by zero, so it has to be finite
        self.k8 = torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.v8 = torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.k_scale = torch.full(shape[:3], 2.0 ** -60, dtype=torch.float32, device=dev)
        self.v_scale = self.k_scale.clone()
        self.page_table = torch.full((self.max_seqs, self.max_pages_per_seq), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.zeros(self.max_seqs, dtype=torch.int32, device=dev)
        self.page_refs = torch.zeros(self.n_pages, dtype=torch.int32, device=dev)
        self.page_uses = torch.zeros(self.n_pages, dtype=torch.int32, device=dev)
        self.scale_uses = torch.zeros((2,) + shape[:3], dtype=torch.int32, device=dev)
        self._workspace = torch.empty(lib.magi_token_cache_workspace_bytes(self.n_pages) // 4, dtype=torch.int32, device=dev)
        c = self._view = TokenCache()
        c.struct_size = C.sizeof(TokenCache)
        for name in sizes:
            setattr(c, name, getattr(self, name))
        for name in ("k8", "v8", "k_scale", "v_scale", "page_table", "seq_lens", "page_refs", "page_uses", "scale_uses"):
            setattr(c, name, getattr(self, name).data_ptr())
        c.workspace = self._workspace.data_ptr()
        self._view_ref = C.byref(c)
        self._attn_bytes = {}  # workspace sizes by call shape

    @property
    def nbytes(self) -> int:
        """Bytes of device memory the cache holds."""
        return sum(t.numel() * t.element_size() for t in (self.k8, self.v8, self.k_scale, self.v_scale, self.page_table,
                                                          self.seq_lens, self.page_refs, self.page_uses, self.scale_uses,
                                                          self._workspace))

    def _entries(self, t, name, n=None):
        t = _index(t, name, self.device, n)
        if t.shape[0] > MAX_ENTRIES:
            raise ValueError(f"{name}: at most {MAX_ENTRIES} entries per call")
        return t

    def reserve(self, seqs: torch.Tensor, n_new: torch.Tensor, stream=None) -> torch.Tensor:
        """Room for n_new[i] more tokens in sequence seqs[i]: takes the pages and advances seq_lens.  Returns the position of
        each entry's first new token (int32; -1 throughout when the call is refused), which append takes as `starts`."""
        seqs = self._entries(seqs, "seqs")
        n_new = self._entries(n_new, "n_new", seqs.shape[0])
        raw = _on(stream, self.device)
        starts = _empty_on(stream, (seqs.shape[0],), torch.int32, self.device)
        check(lib.magi_token_cache_reserve(self.ctx.handle, self._view_ref, seqs.data_ptr(), n_new.data_ptr(), seqs.shape[0],
                                           starts.data_ptr(), raw), self.ctx.handle)
        KERNEL_LAUNCHES[0] += 1
        return starts

    def append(self, layer: int, seqs: torch.Tensor, starts: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               cu_new: Optional[torch.Tensor] = None, max_new: int = 1, stream=None) -> None:
        """Quantise k, v (bf16 [tokens, n_kv_heads, 128], strided) into one layer.  Entry i owns rows cu_new[i]:cu_new[i+1],
        at most max_new of them (cu_new None: one row each), which go to positions starts[i], starts[i]+1, ... of sequence
        seqs[i]; entries with a negative start are skipped.  The scale of a (page, head) is the smallest power of two that
        keeps its finite values within +-448 (and lies in [2^-60, 2^60]); tokens already in the page are re-quantised when
        it grows.  What one reserve gave may be appended in parts, in any order; what an earlier one gave counts as appended
        in every layer once it is in one.  Positions outside the sequence, and pages that other sequences share, are left alone: status E_RANGE."""
        seqs = self._entries(seqs, "seqs")
        starts = self._entries(starts, "starts", seqs.shape[0])
        _rows(k, "k", self.device, self.n_kv_heads), _rows(v, "v", self.device, self.n_kv_heads)
        if k.shape != v.shape:
            raise ValueError("k and v must have the same shape")
        if cu_new is not None:
            cu_new = _index(cu_new, "cu_new", self.device, seqs.shape[0] + 1)
        elif k.shape[0] != seqs.shape[0] or max_new != 1:
            raise ValueError("without cu_new every entry has one token")
        max_new = int(max_new)
        if not 0 <= max_new <= _INT32_MAX:
            raise ValueError("max_new must be a non-negative 32-bit number")
        raw = _on(stream, self.device)
        check(lib.magi_token_cache_append(self.ctx.handle, self._view_ref, _layer(layer, self), seqs.data_ptr(), starts.data_ptr(),
                                          cu_new.data_ptr() if cu_new is not None else None, seqs.shape[0], max_new, k.shape[0],
                                          k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), raw),
              self.ctx.handle)
        KERNEL_LAUNCHES[0] += 1

    def _branch(self, src, dst, share, stream):
        src = self._entries(src, "src")
        dst = self._entries(dst, "dst", src.shape[0])
        raw = _on(stream, self.device)
        check(lib.magi_token_cache_branch(self.ctx.handle, self._view_ref, src.data_ptr(), dst.data_ptr(), src.shape[0], share, raw),
              self.ctx.handle)
        KERNEL_LAUNCHES[0] += 2

    def fork(self, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
        """Make the empty sequences dst[i] continue src[i]: full pages are shared, a last page that is not full is copied.
        A src may repeat; it must not be a dst of the same call."""
        self._branch(src, dst, 1, stream)

    def copy(self, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
        """fork with every page copied, so that nothing is shared."""
        self._branch(src, dst, 0, stream)

    def free(self, seqs: torch.Tensor, stream=None) -> None:
        """Empty the sequences; pages that nobody holds any more become free."""
        seqs = self._entries(seqs, "seqs")
        raw = _on(stream, self.device)
        check(lib.magi_token_cache_free(self.ctx.handle, self._view_ref, seqs.data_ptr(), seqs.shape[0], raw), self.ctx.handle)
        KERNEL_LAUNCHES[0] += 1

    def compact(self, stream=None) -> None:
        """Move the pages in use to the lowest numbers (the i-th one beyond their count to the i-th free one below it) and
        rewrite the tables: afterwards the upper part of every layer's pool is unused."""
        raw = _on(stream, self.device)
        check(lib.magi_token_cache_compact(self.ctx.handle, self._view_ref, raw), self.ctx.handle)
        KERNEL_LAUNCHES[0] += 2


def paged_attn(q: torch.Tensor, cache: TokenPagedKVCache, layer: int, seqs: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
               max_q: int = 1, softmax_scale: Optional[float] = None, causal: bool = True, window: int = 0,
               out: Optional[torch.Tensor] = None, return_lse: bool = True, stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Attention of q (bf16 [tokens, Hq, 128], strided) over the cached sequences, one new token each up to whole prompts.

    Entry i owns query rows cu_q[i]:cu_q[i+1], at most max_q of them (cu_q None: one row each), which stand at the last
    positions of sequence seqs[i] - the new tokens are appended first.  Row at position p sees the cached positions <= p
    (causal) and > p - window (window > 0).  Head h reads kv head h // (Hq // n_kv_heads).  fp32 softmax, the
    weights of V held to 2^-9.4 of each and 2^-29 of the row's largest product of a weight and its page's v_scale; returns
    (out bf16 like q, lse fp32 [tokens, Hq] or None) as chunk_attn does.  A row that sees nothing is zero with lse -inf;
    rows that no entry owns are left as they are in `out` (and undefined in a new one, and in lse).  out may be q itself, or
    memory apart from it (other heads of the same packed tensor, say).  There is no backward pass: the result carries no graph."""
    dev = cache.device
    _rows(q, "q", dev)
    seqs = cache._entries(seqs, "seqs")
    if cu_q is not None:
        cu_q = _index(cu_q, "cu_q", dev, seqs.shape[0] + 1)
    elif q.shape[0] != seqs.shape[0] or max_q != 1:
        raise ValueError("without cu_q every entry has one query row")
    if q.shape[1] % cache.n_kv_heads:
        raise ValueError("the query heads must be a multiple of the cache's kv heads")
    layer, window, max_q = _layer(layer, cache), int(window), int(max_q)
    if not 0 <= window <= _INT32_MAX or not 0 <= max_q <= _INT32_MAX:
        raise ValueError("window and max_q must be non-negative 32-bit numbers")
    if softmax_scale is None:
        scale = 0.0  # the library's default
    else:
        scale = C.c_float(softmax_scale).value  # as the library gets it
        if not 0.0 < scale <= 2e38:
            raise ValueError("softmax_scale must be a positive number that 32 bits hold, at most 2e38")
    raw = _on(stream, dev)
    rows, heads, _ = shape = q.shape
    stride_t, stride_h, _ = q.stride()
    if out is None:
        out = _empty_on(stream, shape, torch.bfloat16, dev)
        out_t, out_h = heads * HEAD_DIM, HEAD_DIM
    else:
        _rows(out, "out", dev, heads)
        if out.shape[0] < rows:
            raise ValueError("out must have at least q's rows")
        _one_place_each(out, "out")
        _itself_or_apart(q, out, "q")
        out_t, out_h, _ = out.stride()
    lse = _empty_on(stream, (rows, heads), torch.float32, dev) if return_lse else None
    handle = cache.ctx.handle
    key = min(max_q, 33), heads  # more than 32 rows: one form
    nbytes = cache._attn_bytes.get(key)
    if nbytes is None:
        nbytes = cache._attn_bytes[key] = lib.magi_paged_attn_workspace_bytes(handle, max_q, heads, cache.n_kv_heads)
    ws = _empty_on(stream, nbytes, torch.uint8, dev)
    p = PagedAttnParams(
        struct_size=_ATTN_BYTES, layer=layer, q=q.data_ptr(), q_stride_t=stride_t, q_stride_h=stride_h, out=out.data_ptr(),
        o_stride_t=out_t, o_stride_h=out_h, lse=lse.data_ptr() if return_lse else None, seqs=seqs.data_ptr(),
        cu_q=cu_q.data_ptr() if cu_q is not None else None, n=seqs.shape[0], total_q=rows, max_q=max_q, n_q_heads=heads,
        softmax_scale=scale, causal=bool(causal), window=window, workspace=ws.data_ptr())
    check(lib.magi_paged_attn_fwd(handle, cache._view_ref, C.byref(p), raw), handle)
    KERNEL_LAUNCHES[0] += 2  # attention and join
    return out, lse


_ROTARY_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_context: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0, device=None
                       ) -> Tuple[torch.Tensor, float]:
    """(inv_freq fp64 [rot_dim/2] on `device` (default: the current CUDA device), mscale) for rotary().  Unscaled: base^(-2i/rot_dim), 1.

    scaling stretches a model's context by `factor`:
      "linear"  every position counts 1/factor
      "ntk"     the base grows to base * factor^(rot_dim / (rot_dim - 2)): the fastest pair keeps its frequency, the slowest
                turns factor times slower
      "yarn"    pairs that turn more than beta_fast times over original_context positions keep their frequency, those that
                turn less than beta_slow times are slowed down by factor, a linear ramp over the pair index between them;
                mscale = 0.1 ln(factor) + 1"""
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be positive and even, got {rot_dim}")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    half, mscale = rot_dim // 2, 1.0
    i = torch.arange(half, dtype=torch.float64)
    if scaling == "ntk" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = float(base) ** (-2.0 * i / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_context <= 0 or not beta_fast > beta_slow > 0:
            raise ValueError("yarn needs original_context > 0 and beta_fast > beta_slow > 0")

        def pair(turns):  # (real) pair index that turns so often over original_context positions
            return rot_dim * math.log(original_context / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        mscale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    return freq.to("cuda" if device is None else device), mscale


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, layout: str = "half", mscale: float = 1.0,
           inverse: bool = False, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Rotary embedding by position of x [tokens, heads, head_dim] (bf16, fp16 or fp32; contiguous last dim, any other strides).

    The first 2 * len(inv_freq) channels of every head are turned by positions[t] * inv_freq[i] (pair i) and multiplied by
    mscale, the others are copied.  layout "half" pairs channels (i, i + half), "interleaved" (2i, 2i + 1).  positions int32
    or int64 [tokens]; inv_freq fp64 (rotary_frequencies).  inverse=True turns backwards: the transposed operator, which maps
    the gradient of the result to the gradient of x.  out may be x itself, or memory apart from it.  No graph is
    recorded: a training step makes the inverse call itself.  qk_norm_rope is the table-driven form of the DiT."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _ROTARY_DTYPES or x.dim() != 3 or (x.shape[2] > 1 and x.stride(2) != 1):
        raise ValueError("x must be a CUDA bf16, fp16 or fp32 [tokens, heads, head_dim] tensor with a contiguous last dim")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    _fit(x, "x")
    dev = x.device
    T, H, D = x.shape
    if not isinstance(positions, torch.Tensor) or positions.device != dev or positions.dtype not in (torch.int32, torch.int64) \
            or positions.dim() != 1 or positions.shape[0] != T or not positions.is_contiguous():
        raise ValueError(f"positions must be a contiguous int32 or int64 tensor of {T} entries on {dev}")
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.device != dev or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 \
            or not inv_freq.is_contiguous() or 2 * inv_freq.shape[0] > D:
        raise ValueError(f"inv_freq must be a contiguous fp64 tensor of at most head_dim / 2 entries on {dev}")
    raw = _on(stream, dev)
    if out is None:
        out = _empty_on(stream, (T, H, D), x.dtype, dev)
    elif out.device != dev or out.dtype != x.dtype or out.shape != x.shape or (D > 1 and out.stride(2) != 1):
        raise ValueError("out must have x's shape, dtype and device and a contiguous last dim")
    else:
        _one_place_each(out, "out")
        _itself_or_apart(x, out, "x")
    if T == 0 or H == 0 or D == 0:
        return out
    (x_t, x_h, _), (out_t, out_h, _) = x.stride(), out.stride()
    p = RotaryParams(
        struct_size=_ROTARY_BYTES, dtype=_ROTARY_DTYPES[x.dtype], x=x.data_ptr(), x_stride_t=x_t, x_stride_h=x_h, out=out.data_ptr(),
        out_stride_t=out_t, out_stride_h=out_h, positions=positions.data_ptr(), positions_are_int64=positions.dtype is torch.int64,
        T=T, H=H, head_dim=D, rot_dim=2 * inv_freq.shape[0], interleaved=layout == "interleaved", inverse=bool(inverse), mscale=mscale,
        inv_freq=inv_freq.data_ptr())
    ctx = Context.get(dev)
    check(lib.magi_rotary_fwd(ctx.handle, C.byref(p), raw), ctx.handle)
    KERNEL_LAUNCHES[0] += 1
    return out
