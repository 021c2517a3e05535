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
    max|x| <= 448 * 2^e. A row with a value that is not finite is stored as
    NaN; an all-zero row has scale 0.
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
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

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

    @property
    def n_pages(self) -> int:
        return self.k.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    def _require(self, op: str) -> None:
        reason = kernels.unavailable_reason(self.k.device)
        if reason is not None:
            raise NotImplementedError(
                f'PagedCache.{op} unavailable on {self.k.device}: {reason}')

    def _index(self, t: torch.Tensor, name: str, shape: tuple) -> None:
        if (t.dtype != torch.int32 or t.device != self.k.device
                or t.dim() != len(shape)
                or any(n is not None and n != m
                       for n, m in zip(shape, t.shape))):
            raise ValueError(f'{name} must be int32 {list(shape)} on '
                             f'{self.k.device}')
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f'{name} must be contiguous in its last '
                             'dimension')

    def _table(self, table: torch.Tensor, n: int) -> None:
        self._index(table, 'table', (n, None))
        if table.shape[1] < 1:
            raise ValueError('a table row holds one page at least')
        if table.shape[1] * self.page_size >= 2 ** 31:
            raise ValueError('a table row addresses fewer than 2^31 rows')
        if n > 1 and table.stride(0) < table.shape[1]:
            raise ValueError('the rows of the table must not overlap')

    def _pack(self, pack: sequences.SequencePack) -> None:
        if pack.device != self.k.device:
            raise ValueError(f'the pack is on {pack.device}, the cache on '
                             f'{self.k.device}')

    def _view(self, table: torch.Tensor) -> tuple:
        """The C ABI's arguments that describe the cache and its table."""
        n, width = table.shape
        return (self.k.data_ptr(), self.v.data_ptr(), _lib.ptr(self.k_scale),
                _lib.ptr(self.v_scale), self.n_pages, self.page_size,
                self.kv_heads, self.head_dim, STORAGE[self.storage][0],
                table.data_ptr(), table.stride(0) if n > 1 else width, width,
                n)

    def write(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
              starts: torch.Tensor, pack: sequences.SequencePack) -> None:
        """Stores packed rows: row i of sequence b becomes row starts[b] + i
        of its context.

        Args:
            k, v: [pack.total_q, kv_heads, D] bf16, contiguous in D (their
                other strides multiples of 8 elements).
            table: [n_sequences, max_pages] int32 page numbers.
            starts: [n_sequences] int32, rows already in each context.
            pack: The rows of each sequence (its q_lengths).
        """
        for name, t in (('k', k), ('v', v)):
            if (t.shape != (pack.total_q, self.kv_heads, self.head_dim)
                    or t.dtype != torch.bfloat16
                    or t.device != self.k.device):
                raise ValueError(
                    f'{name} must be bf16 [{pack.total_q}, {self.kv_heads}, '
                    f'{self.head_dim}] on {self.k.device}')
        self._table(table, pack.n_sequences)
        self._index(starts, 'starts', (pack.n_sequences,))
        self._pack(pack)
        self._require('write')
        k, v = kernels.aligned_rows(k), kernels.aligned_rows(v)
        with torch.cuda.device(self.k.device):
            pack_offsets = kernels.on_stream(pack.q_offsets)
            _lib.call('veda_cache_write', *self._view(table), k.data_ptr(),
                      k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                      v.stride(1), pack.total_q, pack_offsets.data_ptr(),
                      starts.data_ptr(), _lib.stream_ptr(self.k.device))

    def read(self, table: torch.Tensor, pack: sequences.SequencePack
             ) -> tuple[torch.Tensor, torch.Tensor]:
        """The contexts' rows as bf16 (k, v), [pack.total_k, kv_heads, D]:
        rows 0 .. k_lengths[b] - 1 of each sequence, packed."""
        self._table(table, pack.n_sequences)
        self._pack(pack)
        self._require('read')
        shape = (pack.total_k, self.kv_heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=torch.bfloat16,
                            device=self.k.device) for _ in range(2))
        with torch.cuda.device(self.k.device):
            offsets = kernels.on_stream(pack.k_offsets)
            _lib.call('veda_cache_read', *self._view(table),
                      offsets.data_ptr(), pack.total_k, k.data_ptr(),
                      v.data_ptr(), _lib.stream_ptr(self.k.device))
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
                or q.dtype != torch.bfloat16 or q.device != self.k.device):
            raise ValueError(f'q must be bf16 [n_sequences, heads, '
                             f'{self.head_dim}] on {self.k.device}')
        n, heads = q.shape[:2]
        if n < 1 or heads < 1 or heads % self.kv_heads:
            raise ValueError('q needs a sequence, and heads a multiple of '
                             f'{self.kv_heads}')
        if torch.is_grad_enabled() and q.requires_grad:
            raise ValueError('attention over the cache has no gradient')
        self._table(table, n)
        self._index(lengths, 'lengths', (n,))
        scale = kernels.softmax_scale(scale, self.head_dim)
        self._require('attend')
        q = kernels.aligned_rows(q)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = (torch.empty(n, heads, dtype=torch.float32, device=q.device)
               if return_lse else None)
        with torch.cuda.device(self.k.device):
            need = _lib.load().veda_decode_workspace(self.head_dim)
            ws = torch.empty(max(need, 16) // 4, dtype=torch.float32,
                             device=q.device)
            _lib.call('veda_decode', *self._view(table), lengths.data_ptr(),
                      q.data_ptr(), q.stride(0), q.stride(1), heads,
                      out.data_ptr(), _lib.ptr(lse), scale, ws.data_ptr(),
                      ws.numel() * 4, _lib.stream_ptr(q.device))
        return (out, lse) if return_lse else out
