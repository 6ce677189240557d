"""Host-side mirror of the reference's paged KV cache over the C ABI
(crates/izwi-core/src/models/shared/attention/paged.rs): `KvCacheQuantization`, pages appended with
`append_to_pages`, `materialize_pages`, `paged_decode_attention`.  The pool, the page table and the
sequence lengths are device buffers; nothing here computes on the host."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from .ops import Context, _ptr, _stream, _stream_of_device, _workspace_bytes

DEFAULT_KV_PAGE_SIZE = 64                     # paged.rs:10
QUANT = {"none": 0, "int8": 1, "q4_0": 2}


def kv_quantization_from_dtype_hint(dtype: str) -> str:
    """`KvCacheQuantization::from_dtype_hint` (paged.rs:25-36)."""
    d = dtype.strip().lower()
    if d in ("int8", "i8", "q8", "q8_0"):
        return "int8"
    if d in ("q4_0", "q4"):
        return "q4_0"
    return "none"


class PagedKvCache:
    """The K and V pages of `batch` sequences for one layer: every sequence owns `max_pages` pool pages
    (a fixed page table; a serving engine would hand pages out on demand)."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, max_tokens: int, device, quantization: str = "none",
                 page_size: int = DEFAULT_KV_PAGE_SIZE):
        if page_size <= 0:
            raise ValueError("KV page size must be greater than zero")          # append_to_pages, paged.rs:352-356
        self.batch, self.kv_heads, self.head_dim, self.page_size = batch, kv_heads, head_dim, page_size
        self.quantization = quantization
        q = QUANT[quantization]
        self.max_pages = (max_tokens + page_size - 1) // page_size
        n_pages = batch * self.max_pages
        lib = L.lib()
        nbytes, nscales = lib.izb_kv_page_bytes(q, page_size, kv_heads, head_dim), lib.izb_kv_page_scales(q, page_size, kv_heads, head_dim)
        self.k_values = torch.zeros(n_pages * nbytes, device=device, dtype=torch.uint8)
        self.v_values = torch.zeros(n_pages * nbytes, device=device, dtype=torch.uint8)
        self.k_scales = torch.ones(max(n_pages * nscales, 1), device=device, dtype=torch.float32)
        self.v_scales = torch.ones(max(n_pages * nscales, 1), device=device, dtype=torch.float32)
        self.page_table = torch.arange(n_pages, device=device, dtype=torch.int32).reshape(batch, self.max_pages).contiguous()
        self.seq_lens = torch.zeros(batch, device=device, dtype=torch.int32)
        self.max_tokens = self.max_pages * page_size
        self._describe()

    def _describe(self) -> None:
        q = QUANT[self.quantization]
        self._desc = L.KvPages(self.k_values.data_ptr(), self.v_values.data_ptr(), self.k_scales.data_ptr() if q else None,
                               self.v_scales.data_ptr() if q else None, self.page_table.data_ptr(), q, self.page_size, self.kv_heads,
                               self.head_dim, self.max_pages)

    @classmethod
    def view(cls, k_values: torch.Tensor, v_values: torch.Tensor, k_scales: torch.Tensor | None, v_scales: torch.Tensor | None,
             page_table: torch.Tensor, seq_lens: torch.Tensor, kv_heads: int, head_dim: int, quantization: str = "none",
             page_size: int = DEFAULT_KV_PAGE_SIZE) -> "PagedKvCache":
        """A cache over buffers that the caller owns: pools of whole pages (any type, contiguous), their fp32 scales, the
        page table [sequences, max_pages] and the lengths [sequences], both int32.  Several layers may name one table."""
        if page_size <= 0:
            raise ValueError("KV page size must be greater than zero")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or seq_lens.dtype != torch.int32 or seq_lens.shape != page_table.shape[:1]:
            raise ValueError("a page table is int32 [sequences, max_pages], lengths are int32 [sequences]")
        q, lib = QUANT[quantization], L.lib()
        nbytes, nscales = lib.izb_kv_page_bytes(q, page_size, kv_heads, head_dim), lib.izb_kv_page_scales(q, page_size, kv_heads, head_dim)
        tensors = [k_values, v_values, page_table, seq_lens] + ([k_scales, v_scales] if nscales else [])
        if any(t is None or not t.is_cuda or not t.is_contiguous() or t.device != page_table.device for t in tensors):
            raise ValueError("page buffers must be contiguous CUDA tensors of one device")
        pool = k_values.numel() * k_values.element_size()
        if nbytes == 0 or pool % nbytes or v_values.numel() * v_values.element_size() != pool:
            raise ValueError("page pools must hold whole pages, as many for values as for keys")
        if nscales and any(t.dtype != torch.float32 or t.numel() != pool // nbytes * nscales for t in (k_scales, v_scales)):
            raise ValueError("page scales must be fp32, as many as the pool's pages need")
        self = cls.__new__(cls)
        self.batch, self.max_pages = page_table.shape
        self.kv_heads, self.head_dim, self.page_size, self.quantization = kv_heads, head_dim, page_size, quantization
        self.k_values, self.v_values, self.k_scales, self.v_scales = k_values, v_values, k_scales, v_scales
        self.page_table, self.seq_lens = page_table, seq_lens
        self.max_tokens = self.max_pages * page_size
        self._describe()
        return self

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v [batch, n_new, kv_heads, head_dim] bf16 (the reference's `[batch, seq, heads, dim]`)."""
        b, n_new = k.shape[0], k.shape[1]
        assert k.shape == v.shape == (b, n_new, self.kv_heads, self.head_dim) and b == self.batch
        assert k.dtype == v.dtype == torch.bfloat16 and k.is_contiguous() and v.is_contiguous()
        ctx = Context.get(k.device.index)
        row = self.kv_heads * self.head_dim
        L.check(L.lib().izb_kv_pages_append(ctx.handle, _stream(), C.byref(self._desc), _ptr(k), _ptr(v), b, n_new, row, row,
                                            _ptr(self.seq_lens)), "izb_kv_pages_append")
        self.seq_lens += n_new            # on the device, after the append in stream order

    def materialize(self, which: str, max_len: int) -> torch.Tensor:
        """Dense [batch, max_len, kv_heads, head_dim] bf16 copy of the cached keys ("k") or values ("v")."""
        out = torch.zeros(self.batch, max_len, self.kv_heads, self.head_dim, device=self.k_values.device, dtype=torch.bfloat16)
        ctx = Context.get(out.device.index)
        row = self.kv_heads * self.head_dim
        L.check(L.lib().izb_kv_pages_materialize(ctx.handle, _stream(), C.byref(self._desc), 0 if which == "k" else 1, self.batch,
                                                 _ptr(self.seq_lens), _ptr(out), row, max_len * row), "izb_kv_pages_materialize")
        return out

    def decode_attention(self, q: torch.Tensor, scale: float | None = None) -> torch.Tensor:
        """`paged_decode_attention` (paged.rs:578-628): q [batch, heads, head_dim] -> same shape."""
        assert q.dtype == torch.bfloat16 and q.dim() == 3 and q.stride(2) == 1 and q.stride(1) == self.head_dim
        b, h, d = q.shape
        if h % self.kv_heads != 0:
            raise ValueError(f"Paged decode attention received invalid head layout: num_heads={h}, num_kv_heads={self.kv_heads}")
        out = torch.empty(b, h, d, device=q.device, dtype=torch.bfloat16)
        ctx = Context.get(q.device.index)
        need = L.lib().izb_paged_decode_gqa_attention_workspace_bytes(ctx.handle, b, h, self.kv_heads, d, self.max_tokens)
        ws = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
        L.check(L.lib().izb_paged_decode_gqa_attention(ctx.handle, _stream(), _ptr(q), C.byref(self._desc), _ptr(self.seq_lens),
                                                       _ptr(out), b, h, self.max_tokens, q.stride(0), out.stride(0),
                                                       float(d ** -0.5 if scale is None else scale), _ptr(ws), need),
                "izb_paged_decode_gqa_attention")
        return out


def shared_prefix_attention(q: torch.Tensor, prefix: PagedKvCache, suffix: PagedKvCache | None, scale: float | None = None,
                            max_prefix_len: int | None = None, max_seq_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Single-token attention of sequences that share a prompt (izb_shared_prefix_decode_gqa_attention): q
    [groups * n, heads, head_dim] bf16, `prefix` one sequence per group, `suffix` one per row of q, or None.
    Sequence i attends to the whole of prefix i // n and then to its own suffix.  The two bounds (default: what the
    tables hold) size the split over the device; lengths are cut to them."""
    b, h, d = q.shape
    dev, groups, kvh = q.device, prefix.batch, prefix.kv_heads
    q_row, q_head, q_one = q.stride()
    if q.dtype != torch.bfloat16 or not q.is_cuda or q_one != 1 or q_head != d:
        raise ValueError("shared_prefix_attention: q must be bf16 [sequences, heads, head_dim] with dense heads")
    if groups == 0 or b % groups != 0 or d != prefix.head_dim or h % kvh != 0:
        raise ValueError(f"shared_prefix_attention: q {tuple(q.shape)} does not fit {groups} prefixes of {kvh} x {prefix.head_dim}")
    if suffix is not None and (suffix.batch != b or suffix.kv_heads != kvh or suffix.head_dim != d):
        raise ValueError("shared_prefix_attention: the suffix must hold one sequence per query, with the prefix's heads")
    if prefix.page_table.device != dev or (suffix is not None and suffix.page_table.device != dev):
        raise ValueError("shared_prefix_attention: tensors on different devices")
    if out is None:
        out, out_row = torch.empty_like(q, memory_format=torch.contiguous_format), h * d
    else:
        out_row = out.stride(0)
        if out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != dev or out.stride(2) != 1 or out.stride(1) != d:
            raise ValueError("shared_prefix_attention: out must be like q")
    if b == 0:
        return out
    if b == 1:
        q_row = out_row = h * d
    most_p = prefix.max_tokens if max_prefix_len is None else int(max_prefix_len)
    most_s = 0 if suffix is None else suffix.max_tokens if max_seq_len is None else int(max_seq_len)
    ctx = Context.get(dev.index)
    need = _workspace_bytes("izb_shared_prefix_decode_gqa_attention_workspace_bytes", ctx.handle.value, groups, b // groups, h, kvh, d, most_p, most_s)
    ws = torch.empty(need, device=dev, dtype=torch.uint8)
    L.check(L.lib().izb_shared_prefix_decode_gqa_attention(
        ctx.handle, _stream_of_device(dev.index), q.data_ptr(), prefix._desc, prefix.seq_lens.data_ptr(), None if suffix is None else suffix._desc,
        None if suffix is None else suffix.seq_lens.data_ptr(), out.data_ptr(), groups, b // groups, h, most_p, most_s, q_row, out_row,
        d ** -0.5 if scale is None else scale, ws.data_ptr(), need), "izb_shared_prefix_decode_gqa_attention")
    return out


class PagedLayers:
    """The caches of a model's layers for the beams of a search: they share one page table, so that a step's choice
    reorders all of them by one launch (izb_kv_pages_reorder)."""

    def __init__(self, caches: list[PagedKvCache]):
        if not caches:
            raise ValueError("PagedLayers needs at least one cache")
        a = caches[0]
        for c in caches:
            if c.page_table.data_ptr() != a.page_table.data_ptr() or c.page_table.shape != a.page_table.shape:
                raise ValueError("the layers of a PagedLayers must share one page table")
        self.caches, self.batch = caches, a.batch
        self._array = (L.KvPages * len(caches))(*(c._desc for c in caches))

    @classmethod
    def allocate(cls, n_layers: int, sequences: int, kv_heads: int, head_dim: int, max_tokens: int, device, quantization: str = "none",
                 page_size: int = DEFAULT_KV_PAGE_SIZE) -> "PagedLayers":
        """Empty caches of n_layers layers for `sequences` beams of up to max_tokens tokens each."""
        caches = [PagedKvCache(sequences, kv_heads, head_dim, max_tokens, device, quantization, page_size) for _ in range(n_layers)]
        for c in caches[1:]:
            c.page_table = caches[0].page_table
            c._describe()
        return cls(caches)

    def reorder(self, parents: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """Page table under which sequence g * beams + k continues sequence g * beams + parents[g, k]; pages that several
        beams would go on writing are copied.  parents [groups, beams] int32.  The caches go on using the old table until
        `use` is called with the new one."""
        table = self.caches[0].page_table
        if parents.dim() != 2 or parents.dtype != torch.int32 or not parents.is_contiguous() or parents.numel() != self.batch \
                or parents.device != table.device:
            raise ValueError(f"reorder: parents must be contiguous int32 [groups, beams] for {self.batch} sequences")
        if out is None:
            out = torch.empty_like(table)
        elif out.shape != table.shape or out.dtype != torch.int32 or not out.is_contiguous() or out.device != table.device:
            raise ValueError("reorder: out must be like the page table")
        ctx = Context.get(table.device.index)
        L.check(L.lib().izb_kv_pages_reorder(ctx.handle, _stream_of_device(table.device.index), self._array, len(self.caches), parents.data_ptr(), parents.shape[0],
                                             parents.shape[1], self.caches[0].seq_lens.data_ptr(), out.data_ptr()), "izb_kv_pages_reorder")
        return out

    def use(self, table: torch.Tensor) -> None:
        """Makes `table` the page table of all layers."""
        if table.shape != self.caches[0].page_table.shape or table.dtype != torch.int32 or not table.is_contiguous() \
                or table.device != self.caches[0].page_table.device:
            raise ValueError("use: the new page table must be like the old one")
        for i, c in enumerate(self.caches):
            c.page_table = table
            c._desc.page_table = self._array[i].page_table = table.data_ptr()
