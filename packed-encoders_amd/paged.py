"""A paged key/value cache and the calls that use it (``include/pe_paged.h``).

``hip_attention.varlen_attention`` with ``cu_seqlens_k`` attends from new rows to keys that lie in one
packed tensor. Here they lie in pages of a fixed number of tokens, found through a table, so sequences
grow without moving, share the pages of a common prefix, and give them back one by one:

    cache = PagedCache(layers, n_pages, page_size, n_heads_kv, head_dim)
    seq = cache.open()
    cache.extend([seq], [len(prompt)])                   # pages for the new tokens
    table, lens = cache.batch([seq])
    for layer in range(layers):                          # q, k, v of the new tokens, packed
        q = paged_append(k, v, cache.k[layer], cache.v[layer], table, cu_seqlens, lens, q=q, inv_freq=inv_freq)
        out = paged_attention(q, cache.k[layer], cache.v[layer], table, cu_seqlens, lens, max_seqlen)

A call's new tokens are packed like ``varlen_attention``'s queries (``cu_seqlens``) and are the last of
their sequence's ``seqlens_k`` keys. All calls are forward only, run on the current HIP stream and can be
captured into a HIP graph. There is no CPU fallback.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch
from torch import Tensor

from . import _lib
from ._native import native_for
from .hip_rotary import _check_frequencies

_BF16 = torch.bfloat16


def _rows(t: Tensor) -> Tensor:
    """Packed rows [tokens, heads, head_dim] whose rows are 16-byte pieces (a copy where they are not)."""
    fits = (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0)
    return t if fits else t.contiguous()


def _check_cache(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, cu: Tensor, lens: Tensor, device) -> None:
    if k_pages.ndim != 4 or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be [n_pages, page_size, heads, head_dim], alike")
    if k_pages.dtype != _BF16 or v_pages.dtype != _BF16:
        raise ValueError("the paged cache holds bf16")
    if k_pages.shape[1] < _lib.PAGE_MULTIPLE or k_pages.shape[1] % _lib.PAGE_MULTIPLE:
        raise ValueError(f"the page size must be a multiple of {_lib.PAGE_MULTIPLE}, got {k_pages.shape[1]}")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.stride(i) % 8 for i in range(3)):
            raise ValueError(f"{name} needs 16-byte rows: a head_dim stride of 1, other strides multiples of 8")
    if cu.dtype != torch.int32 or cu.ndim != 1 or cu.numel() < 1 or not cu.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous 1-D int32 tensor [n_seq + 1]")
    n_seq = cu.numel() - 1
    if lens.dtype != torch.int32 or lens.shape != (n_seq,) or not lens.is_contiguous():
        raise ValueError("seqlens_k must be a contiguous 1-D int32 tensor [n_seq]")
    if page_table.dtype != torch.int32 or page_table.ndim != 2 or page_table.shape[0] != n_seq:
        raise ValueError("page_table must be an int32 tensor [n_seq, pages]")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table must have a unit stride within a sequence")
    if {t.device for t in (k_pages, v_pages, page_table, cu, lens)} != {device} or device.type != "cuda":
        raise ValueError("the rows, the pages, page_table, cu_seqlens and seqlens_k must be on one HIP device")


def _no_grad(what: str, *tensors: Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} is forward-only; call it under torch.no_grad()")


def _fits(**values: int) -> None:
    for name, x in values.items():
        if not -2**31 <= x < 2**31:
            raise ValueError(f"{name} {x} does not fit 32 bits")


def _on_device(what: str, *tensors: Tensor | None) -> None:
    if any(t is not None and t.device.type == "cpu" for t in tensors):
        raise ValueError(f"{what} runs on the HIP device")


# ----------------------------------------------------------------------------- attention


def _attention_impl(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, cu_seqlens: Tensor,
                    seqlens_k: Tensor, max_seqlen: int, max_seqlen_k: int, softmax_scale: float, window_left: int,
                    window_right: int, causal: bool) -> Tensor:
    _check_cache(k_pages, v_pages, page_table, cu_seqlens, seqlens_k, q.device)
    if q.ndim != 3 or q.dtype != _BF16 or q.shape[2] != k_pages.shape[3]:
        raise ValueError("q must be bf16 [tokens, heads, head_dim] with the pages' head_dim")
    if k_pages.shape[2] < 1 or q.shape[1] < 1 or q.shape[1] % k_pages.shape[2]:
        raise ValueError("query heads must be a multiple of kv heads")
    _fits(tokens=q.shape[0], heads=q.shape[1], max_seqlen=max_seqlen, max_seqlen_k=max_seqlen_k,
          window_left=window_left, window_right=window_right)
    out = torch.empty(q.shape, dtype=_BF16, device=q.device)
    q = _rows(q)
    a = _lib.PagedArgs()
    a.struct_size = ctypes.sizeof(_lib.PagedArgs)
    a.dtype = _lib.DTYPE_BF16
    a.q, a.k_pages, a.v_pages, a.o = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr()
    a.page_table, a.cu_seqlens, a.seqlens_k = page_table.data_ptr(), cu_seqlens.data_ptr(), seqlens_k.data_ptr()
    a.q_stride_token, a.q_stride_head = q.stride(0), q.stride(1)
    a.k_stride_page, a.k_stride_token, a.k_stride_head = k_pages.stride()[:3]
    a.v_stride_page, a.v_stride_token, a.v_stride_head = v_pages.stride()[:3]
    a.o_stride_token, a.o_stride_head = out.stride(0), out.stride(1)
    a.table_stride = page_table.stride(0)
    a.n_seq, a.total_tokens = cu_seqlens.numel() - 1, q.shape[0]
    a.max_seqlen, a.max_seqlen_k = int(max_seqlen), int(max_seqlen_k)
    a.n_heads_q, a.n_heads_kv, a.head_dim = q.shape[1], k_pages.shape[2], q.shape[2]
    a.n_pages, a.page_size, a.max_pages = k_pages.shape[0], k_pages.shape[1], page_table.shape[1]
    a.softmax_scale = float(softmax_scale)
    a.window_left, a.window_right, a.causal = int(window_left), int(window_right), int(causal)
    lib = _lib.library()
    size = ctypes.c_size_t(0)
    _lib.check(lib.pe_paged_workspace_size(ctypes.byref(a), ctypes.byref(size)), "pe_paged_workspace_size")
    workspace = torch.empty(size.value, dtype=torch.uint8, device=q.device) if size.value else None
    with torch.cuda.device(q.device):
        stream = torch.cuda.current_stream(q.device).cuda_stream
        status = lib.pe_paged_attn_fwd(ctypes.byref(a), workspace.data_ptr() if size.value else None, size.value, stream)
    _lib.check(status, "pe_paged_attn_fwd")
    return out


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, cu_seqlens: Tensor,
                    seqlens_k: Tensor, max_seqlen: int, *, max_seqlen_k: int | None = None,
                    softmax_scale: float | None = None, window: tuple[int, int] = (-1, -1),
                    causal: bool = True) -> Tensor:
    """Attention of new tokens over a paged cache: single decoded tokens, drafted ones, chunks of prompts.

    q ``[T, Hq, D]`` bf16 holds the new tokens, packed by int32 ``cu_seqlens``; ``k_pages`` / ``v_pages``
    ``[n_pages, page_size, Hkv, D]`` bf16 hold the keys (any strides that leave rows whole; ``page_size`` a
    multiple of 16), D 64, 128 or 256, Hq a multiple of Hkv. Key j of sequence s is slot ``j % page_size`` of
    page ``page_table[s, j // page_size]`` (int32), and the sequence has ``seqlens_k[s]`` keys (int32), the
    new tokens' own among them: its row r of Lq sits at key position ``seqlens_k[s] - Lq + r``, which
    ``causal`` and ``window`` are measured from as in ``varlen_attention``. A table entry outside
    ``[0, n_pages)`` (-1) maps no page, its keys are masked; a row that reaches no key is zero. What pages
    hold past a sequence's keys, and what masked keys hold, does not matter.

    ``max_seqlen`` bounds every sequence's new tokens, ``max_seqlen_k`` its keys (default: what the table
    holds; a closer bound lets short batches spread better). Returns a new contiguous ``[T, Hq, D]``; rows at
    or beyond ``cu_seqlens[-1]``, and those of a sequence past its bounds or its table, are not written.
    Forward only. Calls of few query rows spread long key ranges over the chip and add the parts in a fixed
    order: results do not change from run to run, but their rounding may with the batch."""
    native = native_for(q)  # first: it serves nothing that the checks below would refuse
    if native is not None and isinstance(k_pages, Tensor) and isinstance(page_table, Tensor):
        held = max_seqlen_k
        if held is None and k_pages.ndim == 4 and page_table.ndim == 2:
            held = min(page_table.shape[1] * k_pages.shape[1], _lib.PAGED_MAX_KEYS)
        scale = q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale
        out = None if held is None else native.paged_attention(
            q, k_pages, v_pages, page_table, cu_seqlens, seqlens_k, max_seqlen, held, scale, window[0], window[1],
            bool(causal))
        if out is not None:
            return out
    _no_grad("paged attention", q, k_pages, v_pages)
    _on_device("paged attention", q, k_pages, v_pages, page_table, cu_seqlens, seqlens_k)
    if page_table.ndim != 2 or k_pages.ndim != 4:
        raise ValueError("page_table must be [n_seq, pages], k_pages [n_pages, page_size, heads, head_dim]")
    if max_seqlen_k is None:
        max_seqlen_k = min(page_table.shape[1] * k_pages.shape[1], _lib.PAGED_MAX_KEYS)
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else float(softmax_scale)
    options = (int(max_seqlen), int(max_seqlen_k), scale, int(window[0]), int(window[1]), bool(causal))
    return torch.ops.pe_hip.paged_attention(q, k_pages, v_pages, page_table, cu_seqlens, seqlens_k, *options)


# ----------------------------------------------------------------------------- new tokens


def _append_impl(q: Tensor | None, k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
                 cu_seqlens: Tensor, seqlens_k: Tensor, inv_freq: Tensor | None, interleaved: bool,
                 rope_scale: float) -> list[Tensor]:
    _check_cache(k_pages, v_pages, page_table, cu_seqlens, seqlens_k, k.device)
    if k.ndim != 3 or k.shape != v.shape or k.dtype != _BF16 or v.dtype != _BF16 or k.shape[1:] != k_pages.shape[2:]:
        raise ValueError("k and v must be bf16 [tokens, heads, head_dim] with the pages' heads and head_dim")
    if v.device != k.device:
        raise ValueError("k and v must be on one device")
    if k.shape[2] % 8 or k.shape[1] < 1:
        raise ValueError("paged_append needs kv heads of a head_dim that is a multiple of 8")
    if q is not None and (q.ndim != 3 or q.dtype != _BF16 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or
                          q.shape[1] < 1 or q.device != k.device):
        raise ValueError("q must be bf16 [tokens, heads, head_dim] beside k")
    _fits(tokens=k.shape[0], heads=k.shape[1], head_dim=k.shape[2], query_heads=0 if q is None else q.shape[1])
    half = 0
    if inv_freq is not None:
        half = _check_frequencies(inv_freq, k.shape[2], k.device)
        inv_freq = inv_freq.contiguous()
    k, v = _rows(k), _rows(v)
    a = _lib.AppendArgs()
    a.struct_size = ctypes.sizeof(_lib.AppendArgs)
    a.dtype = _lib.DTYPE_BF16
    q_out = None
    if q is not None:
        q_out = torch.empty(q.shape, dtype=_BF16, device=q.device)
        q = _rows(q)
        a.q, a.q_out, a.n_heads_q = q.data_ptr(), q_out.data_ptr(), q.shape[1]
        a.q_stride_token, a.q_stride_head = q.stride(0), q.stride(1)
        if q.shape[0] == 0:
            return [q_out]
    a.k, a.v, a.k_pages, a.v_pages = k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    a.page_table, a.cu_seqlens, a.seqlens_k = page_table.data_ptr(), cu_seqlens.data_ptr(), seqlens_k.data_ptr()
    a.inv_freq = inv_freq.data_ptr() if half else None
    a.k_stride_token, a.k_stride_head = k.stride(0), k.stride(1)
    a.v_stride_token, a.v_stride_head = v.stride(0), v.stride(1)
    a.kp_stride_page, a.kp_stride_token, a.kp_stride_head = k_pages.stride()[:3]
    a.vp_stride_page, a.vp_stride_token, a.vp_stride_head = v_pages.stride()[:3]
    a.table_stride = page_table.stride(0)
    a.n_seq, a.total_tokens = cu_seqlens.numel() - 1, k.shape[0]
    a.n_heads_kv, a.head_dim = k.shape[1], k.shape[2]
    a.n_pages, a.page_size, a.max_pages = k_pages.shape[0], k_pages.shape[1], page_table.shape[1]
    a.half, a.interleaved, a.rope_scale = half, int(interleaved), float(rope_scale)
    with torch.cuda.device(k.device):
        stream = torch.cuda.current_stream(k.device).cuda_stream
        _lib.check(_lib.library().pe_paged_append_fwd(ctypes.byref(a), stream), "pe_paged_append_fwd")
    return [] if q_out is None else [q_out]


def paged_append(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, cu_seqlens: Tensor,
                 seqlens_k: Tensor, *, q: Tensor | None = None, inv_freq: Tensor | None = None,
                 interleaved: bool = False, rope_scale: float = 1.0) -> Tensor | None:
    """Write the new tokens' k and v ``[T, Hkv, D]`` (bf16, views of a projection as they are) into the pages,
    in place, each row at its key position (``paged_attention`` says which; ``seqlens_k`` counts the new
    tokens). With ``inv_freq`` k is rotated by that position on the way, as ``rotary`` does (``interleaved``,
    ``rope_scale`` its scale), and so is ``q [T, Hq, D]`` when given: returned as a new contiguous tensor, None
    without q. Without ``inv_freq`` nothing turns and q, when given, is copied.

    Rows whose position is negative or lies in no mapped page are dropped; rows at or beyond
    ``cu_seqlens[-1]`` are left alone (q's too). Sequences that append in one call need last pages of their
    own (``PagedCache`` sees to it). Forward only."""
    native = native_for(k)  # first: it serves nothing that the checks below would refuse
    if native is not None:
        done = native.paged_append(q, k, v, k_pages, v_pages, page_table, cu_seqlens, seqlens_k, inv_freq,
                                   bool(interleaved), rope_scale)
        if done is not None:
            return done if q is not None else None
    _no_grad("paged_append", q, k, v, k_pages, v_pages, inv_freq)
    _on_device("paged_append", q, k, v, k_pages, v_pages, page_table, cu_seqlens, seqlens_k, inv_freq)
    options = (inv_freq, bool(interleaved), float(rope_scale))
    out = torch.ops.pe_hip.paged_append(q, k, v, k_pages, v_pages, page_table, cu_seqlens, seqlens_k, *options)
    return out[0] if q is not None else None


# ----------------------------------------------------------------------------- pages


def _page_bytes(t: Tensor) -> int:
    """Bytes of one page of ``t [..., n_pages, page_size, heads, head_dim]``; ValueError where a page is not
    one dense piece of memory."""
    if t.numel() == 0:
        return 0
    size = 1
    for stride, n in sorted((t.stride(i), t.shape[i]) for i in (-3, -2, -1)):
        if n != 1:
            if stride != size:
                raise ValueError("copy_pages needs pages that are dense in memory")
            size *= n
    return size * t.element_size()


def _copy_impl(pages: list[Tensor], src: list[int], dst: list[int]) -> None:
    if len(src) != len(dst):
        raise ValueError("copy_pages needs as many sources as targets")
    groups: dict[tuple, list[int]] = {}
    for t in pages:
        if t.ndim < 4 or t.device.type != "cuda":
            raise ValueError("copy_pages takes [..., n_pages, page_size, heads, head_dim] tensors on the HIP device")
        if t.device != pages[0].device or t.shape[-4] != pages[0].shape[-4]:
            raise ValueError("copy_pages takes caches of as many pages on one device")
        if t.shape[-4] > 1 and 0 == t.stride(-4) and t.numel():
            raise ValueError("copy_pages needs pages of their own memory")
        key = (t.stride(-4) * t.element_size(), _page_bytes(t))
        bases = groups.setdefault(key, [])
        offsets = [0]
        for n, stride in zip(t.shape[:-4], t.stride()[:-4]):
            offsets = [o + i * stride for o in offsets for i in range(n)]
        if t.numel():
            bases.extend(t.data_ptr() + o * t.element_size() for o in offsets)
    n = len(src)
    n_pages = pages[0].shape[-4] if pages else 0
    targets = set(dst)
    if any(not 0 <= x < n_pages for x in (*src, *dst)):
        raise ValueError(f"copy_pages: page outside [0, {n_pages})")
    if len(targets) != n or not targets.isdisjoint(src):
        raise ValueError("copy_pages: a page is a target once, and then no source")
    if n == 0:
        return
    sources, places = (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst)
    lib = _lib.library()
    with torch.cuda.device(pages[0].device):
        stream = torch.cuda.current_stream(pages[0].device).cuda_stream
        for (stride, size), bases in groups.items():
            _lib.check(lib.pe_copy_pages((ctypes.c_void_p * len(bases))(*bases), len(bases), stride, size, n_pages,
                                         sources, places, n, stream), "pe_copy_pages")


def copy_pages(pages: Tensor | Sequence[Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every cache of ``pages``: a tensor, or several of as many
    pages, ``[..., n_pages, page_size, heads, head_dim]`` of any type, leading axes (layers) each a cache. The
    pairs are host numbers and travel with the launch. A page may be copied to several others, but is the
    target of one pair at most and then no source. ``ValueError`` otherwise, with nothing copied. Every
    page is one dense piece of memory, in 16-byte steps."""
    tensors = [pages] if isinstance(pages, Tensor) else list(pages)
    if not tensors:
        raise ValueError("copy_pages needs a cache")
    native = native_for(tensors[0])  # first: it serves nothing that the checks below would refuse
    if native is not None and native.copy_pages(tensors, src, dst):
        return
    src, dst = [int(x) for x in src], [int(x) for x in dst]
    _no_grad("copy_pages", *tensors)
    _on_device("copy_pages", *tensors)
    torch.ops.pe_hip.copy_pages(tensors, src, dst)


class PagedCache:
    """k and v pages of every layer, ``k[layer]`` and ``v[layer]`` ``[n_pages, page_size, n_heads_kv, head_dim]``, and
    the host's account of which sequence holds which page. A page belongs to the sequences that share it
    and is free when none is left. Calls order their copies on the current stream, like the kernels that
    use the pages; not thread-safe."""

    def __init__(self, layers: int, n_pages: int, page_size: int, n_heads_kv: int, head_dim: int, *,
                 device="cuda", dtype: torch.dtype = _BF16):
        if layers < 1 or n_pages < 1 or page_size < _lib.PAGE_MULTIPLE or page_size % _lib.PAGE_MULTIPLE:
            raise ValueError(f"a cache needs layers, pages and a page size that is a multiple of {_lib.PAGE_MULTIPLE}")
        shape = (layers, n_pages, page_size, n_heads_kv, head_dim)
        self.page_size, self.n_pages = page_size, n_pages
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self._users = [0] * n_pages
        self._free = list(range(n_pages - 1, -1, -1))  # the lowest pages go first
        self._pages: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        """Tokens of a sequence, those reserved by ``extend`` included."""
        return self._lengths[seq]

    def pages(self, seq: int) -> tuple[int, ...]:
        """Its pages in order."""
        return tuple(self._pages[seq])

    def open(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lengths[seq] = [], 0
        return seq

    def fork(self, seq: int) -> int:
        """A sequence of the same tokens, sharing their pages. The first of the two to extend a last page that
        is not full copies it."""
        pages, length = list(self._pages[seq]), self._lengths[seq]
        child = self.open()
        self._pages[child], self._lengths[child] = pages, length
        for page in self._pages[child]:
            self._users[page] += 1
        return child

    def close(self, seq: int) -> None:
        """Give the sequence up; pages that no other shares are free."""
        del self._lengths[seq]
        self._release(self._pages.pop(seq))

    def truncate(self, seq: int, length: int) -> None:
        """Keep the first ``length`` tokens (drafted tokens that were refused)."""
        if not 0 <= length <= self._lengths[seq]:
            raise ValueError(f"cannot truncate {self._lengths[seq]} tokens to {length}")
        keep = -(-length // self.page_size)
        gone = self._pages[seq][keep:]
        del self._pages[seq][keep:]
        self._lengths[seq] = length
        self._release(gone)

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> None:
        """Room for ``counts[i]`` more tokens of each sequence. A last page that is not full and that others
        share is copied first, in every layer. ``MemoryError``, with nothing changed, when the pages left do
        not suffice."""
        seqs, counts = list(seqs), [int(n) for n in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(n < 0 for n in counts):
            raise ValueError("extend takes each sequence once, with a count of new tokens")
        users, need, copied = dict[int, int](), 0, []
        for seq, n in zip(seqs, counts):
            length, held = self._lengths[seq], self._pages[seq]
            need += -(-(length + n) // self.page_size) - len(held)
            if n and length % self.page_size:
                last = held[-1]
                left = users.setdefault(last, self._users[last])
                if left > 1:  # the sequence leaves the page to the others
                    users[last] = left - 1
                    copied.append(seq)
        if need + len(copied) > len(self._free):
            raise MemoryError(f"{need + len(copied)} pages needed, {len(self._free)} free")
        src, dst = [], []
        for seq in copied:
            page = self._take()
            src.append(self._pages[seq][-1])
            dst.append(page)
            self._users[src[-1]] -= 1
            self._pages[seq][-1] = page
        for seq, n in zip(seqs, counts):
            self._lengths[seq] += n
            while len(self._pages[seq]) * self.page_size < self._lengths[seq]:
                self._pages[seq].append(self._take())
        if src:
            copy_pages((self.k, self.v), src, dst)

    def compact(self) -> int:
        """Move the highest pages in use into the lowest free ones until the pages in use are the pool's first;
        returns their number. Tables made before are stale."""
        used = [page for page, n in enumerate(self._users) if n]
        move = dict(zip((p for p in reversed(used) if p >= len(used)), sorted(p for p in self._free if p < len(used))))
        if move:
            copy_pages((self.k, self.v), list(move.keys()), list(move.values()))
            for old, new in move.items():
                self._users[new], self._users[old] = self._users[old], 0
            for held in self._pages.values():
                held[:] = [move.get(page, page) for page in held]
        self._free = list(range(self.n_pages - 1, len(used) - 1, -1))
        return len(used)

    def batch(self, seqs: Sequence[int], *, width: int | None = None) -> tuple[Tensor, Tensor]:
        """``(page_table, seqlens_k)`` of the sequences, on the cache's device: their pages (-1 past them) in
        ``width`` columns (default: as many as the longest needs) and their lengths. One non-blocking copy."""
        longest = max((len(self._pages[s]) for s in seqs), default=0)
        columns = longest if width is None else int(width)
        if columns < longest:
            raise ValueError(f"{longest} pages do not fit a table of {columns} columns")
        host = torch.full((len(seqs) * (columns + 1),), -1, dtype=torch.int32, pin_memory=self.k.is_cuda)
        table, lens = host[:len(seqs) * columns].view(len(seqs), columns), host[len(seqs) * columns:]
        for i, seq in enumerate(seqs):
            table[i, :len(self._pages[seq])] = torch.tensor(self._pages[seq], dtype=torch.int32)
            lens[i] = self._lengths[seq]
        device = host.to(self.k.device, non_blocking=True)
        return device[:len(seqs) * columns].view(len(seqs), columns), device[len(seqs) * columns:]

    def _take(self) -> int:
        page = self._free.pop()
        self._users[page] = 1
        return page

    def _release(self, pages: list[int]) -> None:
        for page in pages:
            self._users[page] -= 1
            if not self._users[page]:
                self._free.append(page)


def _attention_meta(q: Tensor, *args) -> Tensor:
    return torch.empty(q.shape, dtype=_BF16, device=q.device)


def _append_meta(q: Tensor | None, *args) -> list[Tensor]:
    return [] if q is None else [torch.empty(q.shape, dtype=_BF16, device=q.device)]


def _copy_meta(pages: list[Tensor], src: list[int], dst: list[int]) -> None:
    return None


def _register() -> None:
    """Define the ``pe_hip`` operators of this module once per process."""
    lib = torch.library.Library("pe_hip", "FRAGMENT")
    try:
        lib.define("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor cu_seqlens, "
                   "Tensor seqlens_k, int max_seqlen, int max_seqlen_k, float softmax_scale, int window_left, "
                   "int window_right, bool causal) -> Tensor")
        lib.define("paged_append(Tensor? q, Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, "
                   "Tensor page_table, Tensor cu_seqlens, Tensor seqlens_k, Tensor? inv_freq, bool interleaved, "
                   "float rope_scale) -> Tensor[]")
        lib.define("copy_pages(Tensor(a!)[] pages, int[] src, int[] dst) -> ()")
    except RuntimeError:
        return  # already defined by an earlier import in this process
    for name, impl, meta in (("paged_attention", _attention_impl, _attention_meta),
                             ("paged_append", _append_impl, _append_meta), ("copy_pages", _copy_impl, _copy_meta)):
        lib.impl(name, impl, "CUDA")
        lib.impl(name, meta, "Meta")
    globals()["_TORCH_LIBRARY"] = lib


_register()

__all__ = ["PagedCache", "copy_pages", "paged_append", "paged_attention"]
