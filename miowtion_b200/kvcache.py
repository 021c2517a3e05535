"""The paged key-value cache: rows written (and quantised) into pages, whole
contexts read back, and attention of single tokens over it.

    cache = PagedCache.empty(n_pages, 64, kv_heads, 128, 'int8')
    cache.write(k, v, table, starts, pack)     # a prompt's, chunk's or token's
    k_all, v_all = cache.read(table, pack)     # for a chunk behind a context
    out = cache.attend(q, table, lengths)      # one new token per sequence

Row j of sequence b lies in row j % page_size of page table[b, j //
page_size]. Every place and length is read on the device, so the calls run
under a captured graph whose tables and lengths change between replays. A
place outside the table, a page that the cache does not have and a length
that the table row cannot hold touch no memory: the row is skipped (zeros for
a reader, absent for the attention) and the device status word is set, which
`_lib.raise_on_device_status` turns into an error. Pages may be shared by
sequences that only read them; a place that two rows of one call write holds
either of them, or, where rows carry scales, a mixture.

There is no fallback: without a B200 and the built library every call raises.
"""

from __future__ import annotations

import math

import torch

from miowtion_b200 import _lib
from miowtion_b200 import kernels
from miowtion_b200 import sequences

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
# Storage formats: the C ABI's number and the dtype of a code.
STORAGE = {'bf16': (0, torch.bfloat16), 'int8': (1, torch.int8),
           'e4m3': (2, torch.float8_e4m3fn)}


class PagedCache:
    """Pages of keys and values of one layer.

    Args:
        k, v: [n_pages, kv_heads, page_size, D] contiguous, bf16, int8 or
            float8_e4m3fn. D is 64 or 128.
        k_scale, v_scale: [n_pages, kv_heads, page_size] fp32 contiguous for
            int8 and float8_e4m3fn (a row is its codes times its scale), None
            for bf16.

    int8 rows: scale max|x| / 127, codes rounded to nearest (ties to even).
    float8_e4m3fn rows: scale 2^e with the smallest e >= -120 for which
    max|x| <= 448 * 2^e (a value from 1.9375 * 2^127 on rounds to 2^128 and
    reads back as infinity). A row with a value that is not finite is stored
    as NaN; an all-zero row has scale 0.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor,
                 k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError('k and v must be [n_pages, kv_heads, page_size, '
                             'D] of one shape and type')
        names = [n for n, (_, d) in STORAGE.items() if d == k.dtype]
        if not names:
            raise ValueError(f'pages are bf16, int8 or float8_e4m3fn, not '
                             f'{k.dtype}')
        self.storage = names[0]
        n_pages, kv_heads, page_size, dim = k.shape
        if n_pages < 1 or kv_heads < 1:
            raise ValueError('a cache has a page and a head at least')
        if page_size not in PAGE_SIZES:
            raise ValueError(f'page_size must be one of {PAGE_SIZES}: '
                             f'{page_size}')
        if dim not in HEAD_DIMS:
            raise ValueError(f'the head dim must be 64 or 128: {dim}')
        scales = (k_scale, v_scale)
        if self.storage == 'bf16':
            if any(s is not None for s in scales):
                raise ValueError('bf16 pages have no scales')
        elif any(s is None or s.shape != k.shape[:3]
                 or s.dtype != torch.float32 for s in scales):
            raise ValueError(f'{self.storage} pages need fp32 scales '
                             '[n_pages, kv_heads, page_size]')
        tensors = [k, v] + [s for s in scales if s is not None]
        if any(t.device != k.device or not t.is_contiguous()
               or t.data_ptr() % 16 for t in tensors):
            raise ValueError('pages and scales must be contiguous, 16-byte '
                             'aligned and on one device')
        self._tensors = k, v, k_scale, v_scale
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = (
            n_pages, kv_heads, page_size, dim)
        self.device = k.device
        # The C ABI's arguments that describe the pages.
        self._shape = (n_pages, page_size, kv_heads, dim,
                       STORAGE[self.storage][0])
        self._workspace: int | None = None

    @classmethod
    def empty(cls, n_pages: int, page_size: int, kv_heads: int, head_dim: int,
              storage: str = 'bf16', device: torch.device | str = 'cuda'
              ) -> 'PagedCache':
        """A cache of uninitialised pages (nothing reads a row that no call
        has written unless a length covers it)."""
        if storage not in STORAGE:
            raise ValueError(f'storage must be one of {tuple(STORAGE)}: '
                             f'{storage!r}')
        shape = (n_pages, kv_heads, page_size, head_dim)
        dtype = STORAGE[storage][1]
        k, v = (torch.empty(shape, dtype=dtype, device=device)
                for _ in range(2))
        if storage == 'bf16':
            return cls(k, v)
        ks, vs = (torch.empty(shape[:3], device=device) for _ in range(2))
        return cls(k, v, ks, vs)

    # The pages are fixed for the life of the cache (their contents are not).
    @property
    def k(self) -> torch.Tensor:
        return self._tensors[0]

    @property
    def v(self) -> torch.Tensor:
        return self._tensors[1]

    @property
    def k_scale(self) -> torch.Tensor | None:
        return self._tensors[2]

    @property
    def v_scale(self) -> torch.Tensor | None:
        return self._tensors[3]

    def _index(self, t: torch.Tensor, name: str, n: int) -> int:
        """Address of an int32 [n] argument."""
        if (t.dtype != torch.int32 or t.shape != (n,)
                or t.device != self.device):
            raise ValueError(f'{name} must be int32 [{n}] on {self.device}')
        if n > 1 and t.stride(0) != 1:
            raise ValueError(f'{name} must be contiguous')
        return t.data_ptr()

    def _view(self, table: torch.Tensor, n: int) -> tuple:
        """The C ABI's arguments that describe the cache and its table of n
        sequences."""
        if (table.dtype != torch.int32 or table.dim() != 2
                or table.shape[0] != n or table.device != self.device):
            raise ValueError(f'table must be int32 [{n}, max_pages] on '
                             f'{self.device}')
        width = table.shape[1]
        if width < 1:
            raise ValueError('a table row holds one page at least')
        if width * self.page_size >= 2 ** 31:
            raise ValueError('a table row addresses fewer than 2^31 rows')
        pitch, step = table.stride()
        if width > 1 and step != 1:
            raise ValueError('table must be contiguous in its last dimension')
        if n == 1:
            pitch = width
        elif pitch < width:
            raise ValueError('the rows of the table must not overlap')
        k, v, k_scale, v_scale = self._tensors
        return (k.data_ptr(), v.data_ptr(), _lib.ptr(k_scale),
                _lib.ptr(v_scale), *self._shape, table.data_ptr(), pitch,
                width, n)

    def _pack(self, pack: sequences.SequencePack) -> None:
        if pack.device != self.device:
            raise ValueError(f'the pack is on {pack.device}, the cache on '
                             f'{self.device}')

    def write(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
              starts: torch.Tensor, pack: sequences.SequencePack) -> None:
        """Stores packed rows: row i of sequence b becomes row starts[b] + i
        of its context.

        Args:
            k, v: [pack.total_q, kv_heads, D] bf16, contiguous in D (their
                other strides multiples of 8 elements), without gradients.
            table: [n_sequences, max_pages] int32 page numbers.
            starts: [n_sequences] int32, rows already in each context.
            pack: The rows of each sequence (its q_lengths).
        """
        rows = (pack.total_q, self.kv_heads, self.head_dim)
        for name, t in (('k', k), ('v', v)):
            if (t.shape != rows or t.dtype != torch.bfloat16
                    or t.device != self.device):
                raise ValueError(f'{name} must be bf16 {list(rows)} on '
                                 f'{self.device}')
        if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
            raise ValueError('rows of the cache carry no gradient: write them '
                             'under torch.no_grad() or detached')
        kernels.refuse_tangents('PagedCache.write', k, v)
        view = self._view(table, pack.n_sequences)
        start_args = self._index(starts, 'starts', pack.n_sequences)
        self._pack(pack)
        kernels.require_ready(self.device, 'PagedCache.write')
        k, v = kernels.aligned_rows(k), kernels.aligned_rows(v)
        (k_row, k_head, _), (v_row, v_head, _) = k.stride(), v.stride()
        _lib.call_on(self.device.index, 'veda_cache_write', *view,
                     k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head,
                     rows[0], pack.offsets()[0].data_ptr(), start_args)

    def read(self, table: torch.Tensor, pack: sequences.SequencePack
             ) -> tuple[torch.Tensor, torch.Tensor]:
        """The contexts' rows as bf16 (k, v), [pack.total_k, kv_heads, D]:
        rows 0 .. k_lengths[b] - 1 of each sequence, packed."""
        view = self._view(table, pack.n_sequences)
        self._pack(pack)
        kernels.require_ready(self.device, 'PagedCache.read')
        k, v = (torch.empty((pack.total_k, self.kv_heads, self.head_dim),
                            dtype=torch.bfloat16, device=self.device)
                for _ in range(2))
        _lib.call_on(self.device.index, 'veda_cache_read', *view,
                     pack.offsets()[1].data_ptr(), pack.total_k, k.data_ptr(),
                     v.data_ptr())
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor,
               lengths: torch.Tensor, scale: float | None = None,
               return_lse: bool = False):
        """Attention of one query per sequence over its cached rows.

        Args:
            q: [n_sequences, heads, D] bf16, heads a multiple of kv_heads
                (head h reads kv head h // (heads // kv_heads)).
            table: [n_sequences, max_pages] int32 page numbers.
            lengths: [n_sequences] int32, rows of each context to attend to
                (the new token's own row among them, once it is written).
            scale: Softmax scale; None for D ** -0.5.
            return_lse: Also return the [n_sequences, heads] fp32
                log-sum-exp.

        Returns:
            out [n_sequences, heads, D] bf16 (and lse); 0 and -inf for a
            sequence without rows.
        """
        if (q.dim() != 3 or q.shape[2] != self.head_dim
                or q.dtype != torch.bfloat16 or q.device != self.device):
            raise ValueError(f'q must be bf16 [n_sequences, heads, '
                             f'{self.head_dim}] on {self.device}')
        n, heads, dim = q.shape
        if n < 1 or heads < 1 or heads % self.kv_heads:
            raise ValueError('q needs a sequence, and heads a multiple of '
                             f'{self.kv_heads}')
        if q.requires_grad and torch.is_grad_enabled():
            raise ValueError('attention over the cache has no gradient')
        kernels.refuse_tangents('PagedCache.attend', q)
        view = self._view(table, n)
        length_args = self._index(lengths, 'lengths', n)
        scale = kernels.softmax_scale(scale, dim)
        kernels.require_ready(self.device, 'PagedCache.attend')
        q = kernels.aligned_rows(q)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = (q.new_empty((n, heads), dtype=torch.float32) if return_lse
               else None)
        if self._workspace is None:
            with torch.cuda.device(self.device):
                self._workspace = _lib.load().veda_decode_workspace(dim)
        # Allocated for the call: captured graphs share no workspace.
        ws = q.new_empty((self._workspace // 4,), dtype=torch.float32)
        q_row, q_head, _ = q.stride()
        _lib.call_on(self.device.index, 'veda_decode', *view, length_args,
                     q.data_ptr(), q_row, q_head, heads, out.data_ptr(),
                     _lib.ptr(lse), scale, ws.data_ptr(), self._workspace)
        return (out, lse) if return_lse else out
