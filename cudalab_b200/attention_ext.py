"""Extension objects of the operators between a decoder layer's projections:
per-head norm and rotation of q and k, the quantised paged KV cache, and
attention over it.  No counterpart in the reference, whose operators end at
the projections; the checks run here before any device work, in the order of
the arguments, and raise RuntimeError.  The computation always goes through
the C ABI of libcudalab_gemv.so, on the current stream of the tensors' device.

Common call: the torch binding (csrc/torch_fast.cpp) checks the tensors in C++
and calls the C ABI; a call it declines takes the ordered checks below.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as nat
from .ext import _binding, _chk, _stream_ptr

_TYPES = {torch.float16: nat.CL_DTYPE_F16, torch.bfloat16: nat.CL_DTYPE_BF16}
HEAD_DIMS = (64, 128, 256)
BLOCK = 16  # tokens of a cache block


def block_bytes(head_dim: int, bits: int) -> int:
    """Bytes of one block: 16 K rows, 16 V rows and their 32 fp16 scales."""
    return 4 * head_dim * bits + 64


class _Ext:
    kind = ""

    def __init__(self) -> None:
        self._lib = nat.load()
        self._tb = _binding()

    def _call(self, fn, dev: torch.device, *args) -> None:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream_ptr(dev))
        if rc != nat.CL_OK:
            raise RuntimeError(f"{self.kind} launch failed ({rc}): {nat.last_error(self._lib)}")


def _rows(name: str, x: torch.Tensor, dims: int, like: torch.Tensor | None = None) -> None:
    """A tensor of 16-bit rows whose last dimension is contiguous."""
    _chk(x.dim() == dims, f"{name} must be {dims}-D, got {x.dim()}-D")
    _chk(x.dtype in _TYPES, f"{name} must be float16 or bfloat16, got {x.dtype}")
    if like is not None:
        _chk(x.dtype == like.dtype, f"{name} must be {like.dtype}, got {x.dtype}")
    _chk(x.stride(-1) == 1 or x.size(-1) == 1, f"the last dimension of {name} must be contiguous")
    _chk(x.is_cuda, f"{name} must be a CUDA tensor")
    if like is not None:
        _chk(x.device == like.device, f"{name} must be on {like.device}, got {x.device}")


def _plain(name: str, x: torch.Tensor, dims: int, dtypes, dev: torch.device) -> None:
    """A contiguous tensor of one of `dtypes` on `dev`."""
    _chk(x.dim() == dims, f"{name} must be {dims}-D, got {x.dim()}-D")
    _chk(x.dtype in dtypes, f"{name} must be {' or '.join(map(str, dtypes))}, got {x.dtype}")
    _chk(x.is_contiguous(), f"{name} must be contiguous")
    _chk(x.device == dev, f"{name} must be on {dev}, got {x.device}")


def _apart(name: str, x: torch.Tensor) -> None:
    """An output whose elements do not share memory: each dimension steps past all that the
    ones of smaller strides span (an expanded tensor's, or an overlapping window's, does not)."""
    end = 0  # last element of the dimensions so far
    for step, n in sorted((s, n) for n, s in zip(x.shape, x.stride()) if n > 1):
        _chk(x.numel() == 0 or step > end, f"{name} must not overlap itself")
        end += (n - 1) * step


def _separate(name: str, y: torch.Tensor, other: str, x: torch.Tensor) -> None:
    """An output whose memory lies outside an input's first to last element."""
    def ends(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if x.numel() and y.numel():
        (a, b), (c, d) = ends(y), ends(x)
        _chk(b <= c or d <= a, f"{name} must not overlap {other}")


def _pages(pages: torch.Tensor, head_dim: int, dev: torch.device | None = None) -> tuple:
    """(bits, page_size) of a cache tensor for heads of head_dim elements."""
    _chk(head_dim in HEAD_DIMS, f"head_dim must be 64, 128 or 256, got {head_dim}")
    _chk(pages.dim() == 4, f"pages must be 4-D [pages, kv_heads, page_size / 16, block bytes], "
                           f"got {pages.dim()}-D")
    _chk(pages.dtype == torch.uint8, f"pages must be uint8, got {pages.dtype}")
    bits = {block_bytes(head_dim, b): b for b in (8, 4)}.get(pages.size(3))
    _chk(bits is not None, f"pages has blocks of {pages.size(3)} bytes; head_dim {head_dim} needs "
                           f"{block_bytes(head_dim, 8)} (int8) or {block_bytes(head_dim, 4)} (int4)")
    _chk(pages.numel() > 0, "pages must not be empty")
    _chk(pages.is_contiguous(), "pages must be contiguous")
    _chk(pages.is_cuda, "pages must be a CUDA tensor")
    _chk(dev is None or pages.device == dev, f"pages must be on {dev}, got {pages.device}")
    return bits, pages.size(2) * BLOCK


class QkNormRopeExt(_Ext):
    """RMSNorm of every head of q and k, and the rotation by position, in one pass."""
    kind = "qknorm_rope"

    def _validate(self, q, k, q_weight, k_weight, table, positions, eps) -> None:
        _rows("q", q, 3)
        _rows("k", k, 3, q)
        T, Hq, D = q.shape
        _chk(k.size(0) == T and k.size(2) == D,
             f"k must be [{T}, kv_heads, {D}], got {list(k.shape)}")
        _chk(Hq > 0 and k.size(1) > 0, "q and k must have at least one head")
        _chk(D % 16 == 0 and 0 < D <= 256, f"head_dim must be a multiple of 16 up to 256, got {D}")
        _chk((q_weight is None) == (k_weight is None),
             "q_weight and k_weight must both be given, or neither")
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is not None:
                _plain(name, w, 1, (q.dtype,), q.device)
                _chk(w.size(0) == D, f"{name} must have {D} elements, got {w.size(0)}")
        _plain("table", table, 2, (torch.float32,), q.device)
        R = table.size(1)
        _chk(R % 16 == 0 and 0 < R <= D,
             f"table must have a multiple of 16 up to head_dim={D} columns, got {R}")
        _chk(table.size(0) > 0, "table must have at least one row")
        _chk(table.data_ptr() % 16 == 0, "table must be 16-byte aligned")
        _plain("positions", positions, 1, (torch.int64, torch.int32), q.device)
        _chk(positions.size(0) == T, f"positions must have {T} elements, got {positions.size(0)}")
        _chk(eps >= 0.0 and eps != float("inf"), f"eps must be finite and >= 0, got {eps}")

    def _launch(self, q, k, q_weight, k_weight, table, positions, q_out, k_out, eps, interleaved):
        d = nat.QkNormRopeDesc(
            q.size(0), table.size(0), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
            q_out.stride(0), q_out.stride(1), k_out.stride(0), k_out.stride(1), q.size(1),
            k.size(1), q.size(2), table.size(1), int(interleaved),
            int(positions.dtype == torch.int64), _TYPES[q.dtype], eps)
        self._call(self._lib.cl_qknorm_rope, q.device, q.data_ptr(), k.data_ptr(),
                   None if q_weight is None else q_weight.data_ptr(),
                   None if k_weight is None else k_weight.data_ptr(), table.data_ptr(),
                   positions.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), ctypes.byref(d))

    def forward(self, q, k, q_weight, k_weight, table, positions, eps: float = 1e-6,
                interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
        """q [tokens, q_heads, head_dim], k [tokens, kv_heads, head_dim] (any strides but a
        contiguous last dimension, e.g. slices of one fused projection), weights [head_dim]
        (None, None: rotation alone), table fp32 [rows, rotary] (rotary / 2 cosines, then the
        sines), positions int64 / int32 [tokens] -> contiguous (q, k).  Elements past `rotary`
        are normalised and not turned; interleaved: pairs (2i, 2i + 1) instead of
        (i, i + rotary / 2)."""
        if self._tb is not None:
            r = self._tb.qknorm_rope(q, k, q_weight, k_weight, table, positions, eps, interleaved)
            if r is not None:
                return r
        self._validate(q, k, q_weight, k_weight, table, positions, eps)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        self._launch(q, k, q_weight, k_weight, table, positions, q_out, k_out, eps, interleaved)
        return q_out, k_out

    def forward_into(self, q, k, q_weight, k_weight, table, positions, q_out, k_out,
                     eps: float = 1e-6, interleaved: bool = False) -> None:
        """Same into q_out, k_out, which may be q and k themselves."""
        self._validate(q, k, q_weight, k_weight, table, positions, eps)
        for name, y, x in (("q_out", q_out, q), ("k_out", k_out, k)):
            _rows(name, y, 3, x)
            _chk(y.shape == x.shape, f"{name} must be {list(x.shape)}, got {list(y.shape)}")
            _apart(name, y)
        self._launch(q, k, q_weight, k_weight, table, positions, q_out, k_out, eps, interleaved)


class KvCacheExt(_Ext):
    """The quantised paged cache: tokens are quantised as they are written (int8 or int4, one
    fp16 scale per token and head) and can be read back.  Token slot = page * page_size +
    offset in the page."""
    kind = "kvcache"

    @staticmethod
    def empty(num_pages: int, kv_heads: int, head_dim: int, bits: int = 8, page_size: int = 64,
              device="cuda") -> torch.Tensor:
        """A cache tensor uint8 [num_pages, kv_heads, page_size / 16, block bytes] (zeros)."""
        _chk(head_dim in HEAD_DIMS, f"head_dim must be 64, 128 or 256, got {head_dim}")
        _chk(bits in (8, 4), f"bits must be 8 or 4, got {bits}")
        _chk(page_size > 0 and page_size % BLOCK == 0,
             f"page_size must be a multiple of 16, got {page_size}")
        _chk(num_pages > 0 and kv_heads > 0, "num_pages and kv_heads must be > 0")
        return torch.zeros(num_pages, kv_heads, page_size // BLOCK, block_bytes(head_dim, bits),
                           dtype=torch.uint8, device=device)

    def _desc(self, k, v, pages, bits, page_size):
        return nat.KvCacheDesc(k.size(0), pages.size(0), k.stride(0), k.stride(1), v.stride(0),
                               v.stride(1), pages.size(1), k.size(2), bits, page_size,
                               _TYPES[k.dtype])

    def _validate(self, k, v, pages, slots) -> tuple:
        _rows("k", k, 3)
        _rows("v", v, 3, k)
        _chk(v.shape == k.shape, f"v must be {list(k.shape)}, got {list(v.shape)}")
        form = _pages(pages, k.size(2), k.device)
        _chk(k.size(1) == pages.size(1),
             f"k and v must have the cache's {pages.size(1)} heads, got {k.size(1)}")
        _plain("slots", slots, 1, (torch.int64,), k.device)
        _chk(slots.size(0) == k.size(0),
             f"slots must have {k.size(0)} elements, got {slots.size(0)}")
        return form

    def write(self, k, v, pages, slots) -> None:
        """Quantises k, v [tokens, kv_heads, head_dim] into their slots (int64 [tokens], no two
        the same; negative: the token is skipped)."""
        if self._tb is not None and self._tb.kvcache_write(k, v, pages, slots):
            return
        bits, page_size = self._validate(k, v, pages, slots)
        self._call(self._lib.cl_kvcache_write, k.device, k.data_ptr(), v.data_ptr(),
                   pages.data_ptr(), slots.data_ptr(),
                   ctypes.byref(self._desc(k, v, pages, bits, page_size)))

    def read(self, pages, slots, head_dim: int, dtype=torch.float16) -> tuple:
        """(k, v) [tokens, kv_heads, head_dim] of the slots; zeros for a negative slot."""
        if self._tb is not None:
            r = self._tb.kvcache_read(pages, slots, head_dim, dtype is torch.bfloat16) \
                if dtype in _TYPES else None
            if r is not None:
                return r
        _chk(dtype in _TYPES, f"dtype must be float16 or bfloat16, got {dtype}")
        _pages(pages, head_dim)
        _plain("slots", slots, 1, (torch.int64,), pages.device)
        shape = (slots.size(0), pages.size(1), head_dim)
        k = torch.empty(shape, dtype=dtype, device=pages.device)
        v = torch.empty(shape, dtype=dtype, device=pages.device)
        self.read_into(pages, slots, k, v)
        return k, v

    def read_into(self, pages, slots, k, v) -> None:
        """Same into k, v (float16 or bfloat16, any strides but a contiguous last dimension)."""
        bits, page_size = self._validate(k, v, pages, slots)
        _apart("k", k)
        _apart("v", v)
        self._call(self._lib.cl_kvcache_read, k.device, pages.data_ptr(), slots.data_ptr(),
                   k.data_ptr(), v.data_ptr(),
                   ctypes.byref(self._desc(k, v, pages, bits, page_size)))


class KvAttentionExt(_Ext):
    """Attention of the new tokens of each sequence over its cached tokens."""
    kind = "kvattention"

    def __init__(self) -> None:
        super().__init__()
        n = ctypes.c_size_t(0)
        self._lib.cl_kvattention_workspace(ctypes.byref(n))
        self.workspace_bytes = n.value

    def workspace(self, device="cuda") -> torch.Tensor:
        """Scratch for `workspace=`: kept by the caller and used by one call at a time (calls
        that may overlap, on other streams, need their own)."""
        return torch.zeros(self.workspace_bytes, dtype=torch.uint8, device=device)

    def _validate(self, q, pages, page_table, lengths, scale, window) -> tuple:
        _chk(q.dim() in (3, 4), f"q must be [batch, heads, head_dim] or [batch, new_tokens, heads, "
                                f"head_dim], got {q.dim()}-D")
        _rows("q", q, q.dim())
        B, Hq, D = q.size(0), q.size(-2), q.size(-1)
        form = _pages(pages, D, q.device)
        _chk(q.dim() == 3 or q.size(1) > 0, "q must have at least one new token")
        _chk(Hq > 0 and Hq % pages.size(1) == 0,
             f"the {Hq} heads of q must be a multiple of the cache's {pages.size(1)}")
        _chk(B <= 4096, f"at most 4096 sequences, got {B}")
        _plain("lengths", lengths, 1, (torch.int32,), q.device)
        _chk(lengths.size(0) == B, f"lengths must have {B} elements, got {lengths.size(0)}")
        _chk(page_table.dim() == 2 and page_table.size(0) == B,
             f"page_table must be [{B}, pages], got {list(page_table.shape)}")
        _chk(page_table.dtype == torch.int32, f"page_table must be int32, got {page_table.dtype}")
        _chk(page_table.size(1) <= 1 or page_table.stride(1) == 1,
             "the rows of page_table must be contiguous")
        _chk(page_table.device == q.device, f"page_table must be on {q.device}")
        _chk(window >= 0, f"window must be >= 0, got {window}")
        _chk(scale is None or (scale == scale and abs(scale) != float("inf")),
             f"scale must be finite, got {scale}")
        return form

    def _forward(self, q, pages, page_table, lengths, scale, window, workspace, prefix_pages,
                 prefix_length, out, return_lse):
        bits, page_size = self._validate(q, pages, page_table, lengths, scale, window)
        dev, D = q.device, q.size(-1)
        if workspace is None:
            workspace = self.workspace(dev)
        _plain("workspace", workspace, 1, (torch.uint8,), dev)
        _chk(workspace.numel() >= self.workspace_bytes and workspace.data_ptr() % 16 == 0,
             f"workspace must have {self.workspace_bytes} bytes, 16-byte aligned")
        n_prefix = 0
        if prefix_length:
            _chk(prefix_pages is not None, f"prefix_length is {prefix_length}: prefix_pages must "
                                           "be given")
            _plain("prefix_pages", prefix_pages, 1, (torch.int32,), dev)
            n_prefix = prefix_pages.size(0)
            _chk(0 <= prefix_length <= n_prefix * page_size,
                 f"prefix_length must be in [0, {n_prefix * page_size}], got {prefix_length}")
            _chk(window == 0, "a prefix and a window exclude each other")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        else:
            _chk(out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
                 and out.device == dev and out.data_ptr() % 16 == 0,
                 f"out must be contiguous {q.dtype} {list(q.shape)} on {dev}, 16-byte aligned")
            _separate("out", out, "q", q)  # rows are written while others are still read
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev) if return_lse else None
        q4 = q.unsqueeze(1) if q.dim() == 3 else q
        if prefix_length and q4.size(0) > 1 and q4.size(1) > 1 \
                and q4.stride(0) != q4.size(1) * q4.stride(1):
            q4 = q4.contiguous()
        d = nat.KvAttentionDesc(
            pages.size(0), page_table.stride(0), q4.stride(0), q4.stride(1), q4.stride(2),
            q4.size(0), q4.size(1), q4.size(2), pages.size(1), D, bits, page_size,
            page_table.size(1), int(window), _TYPES[q.dtype], int(prefix_length), n_prefix,
            D ** -0.5 if scale is None else float(scale))

        scratch = None
        if prefix_length:
            n = ctypes.c_size_t(0)
            rc = self._lib.cl_kvattention_prefix_floats(ctypes.byref(d), ctypes.byref(n))
            if rc != nat.CL_OK:
                raise RuntimeError(f"{self.kind} failed ({rc}): {nat.last_error(self._lib)}")
            scratch = torch.empty(n.value, dtype=torch.float32, device=dev)

        def ptr(x):
            return None if x is None else x.data_ptr()

        self._call(self._lib.cl_kvattention, dev, q4.data_ptr(), pages.data_ptr(),
                   page_table.data_ptr(), lengths.data_ptr(),
                   ptr(prefix_pages) if prefix_length else None, out.data_ptr(), ptr(lse),
                   ptr(scratch), workspace.data_ptr(), ctypes.byref(d))
        return (out, lse) if return_lse else out

    def forward(self, q, pages, page_table, lengths, scale: float | None = None, window: int = 0,
                workspace=None, return_lse: bool = False):
        """q [batch, heads, head_dim] (one new token per sequence) or [batch, new_tokens, heads,
        head_dim]; page_table int32 [batch, pages], lengths int32 [batch] (the new tokens
        included, already written to the cache).  Row i sees its sequence up to its own token,
        with window > 0 the last `window` tokens of that.  Heads / cache heads grouped; scale
        None: head_dim ** -0.5.  -> out like q (contiguous), with return_lse also the natural log
        of the softmax's denominator, fp32.  A row that sees nothing gives zeros and -inf."""
        if self._tb is not None and workspace is not None:
            r = self._tb.kvattention(q, pages, page_table, lengths, None, 0,
                                     0.0 if scale is None else scale, scale is None, window,
                                     workspace, return_lse)
            if r is not None:
                return r
        return self._forward(q, pages, page_table, lengths, scale, window, workspace, None, 0,
                             None, return_lse)

    def forward_into(self, q, pages, page_table, lengths, out, scale: float | None = None,
                     window: int = 0, workspace=None) -> None:
        """Same into `out` (contiguous, like q, apart from it)."""
        self._forward(q, pages, page_table, lengths, scale, window, workspace, None, 0, out, False)

    def forward_shared(self, q, pages, prefix_pages, prefix_length: int, page_table, lengths,
                       scale: float | None = None, workspace=None, return_lse: bool = False):
        """forward for a batch whose sequences all begin with the same prefix_length tokens, held
        by prefix_pages (int32); page_table and lengths cover each sequence's own tokens after
        them.  The prefix is read once for the whole batch."""
        _chk(prefix_length >= 0, f"prefix_length must be >= 0, got {prefix_length}")
        if self._tb is not None and workspace is not None:
            r = self._tb.kvattention(q, pages, page_table, lengths, prefix_pages, prefix_length,
                                     0.0 if scale is None else scale, scale is None, 0, workspace,
                                     return_lse)
            if r is not None:
                return r
        return self._forward(q, pages, page_table, lengths, scale, 0, workspace, prefix_pages,
                             prefix_length, None, return_lse)
