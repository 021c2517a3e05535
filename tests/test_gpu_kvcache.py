"""The paged cache on the GPU against its definition in 64 bits.

Codes and scales have to be equal, and rows read back are code * scale rounded
once. The attention's bound counts its roundings, elementwise: weights to the
16-bit type of the products (half a step: 2^-8 bf16, 2^-11 fp16 for int8 and
e4m3 pages) and the output to bf16 (2^-8),
    |out - want| <= (w + 2 s) sum_j p_j |v_j| + 2^-8 |want|
                    + 2^-14 sum_j p_j |v_j|,
the last term for fp32 sums and exponentials and for q's elements below
2^-14 of their head's largest. s is what the fp32 scores may be off: a sum of
D products of total size A = scale max_j sum_d |q_d k_jd|, then three
factors, is off by (D + 8) 2^-24 A, which is a relative error of a weight and
again of the weights' sum (scores of a few thousand make it 2^-12). The
log-sum-exp is fp32 throughout: s and the exponentials' 2^-22.
"""

import math

import numpy as np
import pytest
import torch

from miowtion_b200 import _lib
from miowtion_b200 import kvcache
from miowtion_b200 import sequences

pytestmark = pytest.mark.gpu

DEV = 'cuda'
STORAGES = ['bf16', 'int8', 'e4m3']


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.device_status(reset=True)
    yield
    assert _lib.device_status(reset=True) == 0, 'the status word was set'


def rows(n, heads, dim, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=gen) * scale
    return x.to(torch.bfloat16).to(DEV)


def codes64(x, storage):
    """(codes, scales) of bf16 rows in real arithmetic (fp64 numpy)."""
    x = x.double().cpu().numpy()
    top = np.abs(x).max(-1, keepdims=True)
    if storage == 'int8':
        codes = np.round(np.divide(x * 127, top, where=top > 0,
                                   out=np.zeros_like(x)))
        scale = (top.astype(np.float32) / np.float32(127)).astype(np.float64)
    else:
        e = np.full(top.shape, -120.0)
        while (top > 448 * 2.0 ** e).any():
            e = np.where(top > 448 * 2.0 ** e, e + 1, e)
        y = x / 2.0 ** e
        power = np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6)))
        step = 2.0 ** (power - 3)
        codes = np.round(y / step) * step
        scale = np.where(top > 0, 2.0 ** e, 0.0)
    return codes, scale[..., 0]


def table_of(counts, extra, seed):
    """Pages in any order; unused entries name no page."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(counts) + extra
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(counts), max(max(counts), 1)), -1,
                       dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEV), max(total, 1)


def poison(cache):
    """Pages nothing has written hold NaN (int8: the scales do)."""
    for t in (cache.k, cache.v):
        if t.dtype == torch.int8:
            t.fill_(-128)
        else:
            t.view(torch.uint8).fill_(0xff)
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(math.nan)


def filled(storage, contexts, size, heads, dim, seed, extra=2):
    counts = [-(-c // size) for c in contexts]
    table, total = table_of(counts, extra, seed)
    cache = kvcache.PagedCache.empty(total, size, heads, dim, storage, DEV)
    poison(cache)
    pack = sequences.SequencePack(contexts, device=DEV)
    k = rows(pack.total_k, heads, dim, seed + 1)
    v = rows(pack.total_k, heads, dim, seed + 2)
    starts = torch.zeros(len(contexts), dtype=torch.int32, device=DEV)
    cache.write(k, v, table, starts, pack)
    return cache, table, pack, k, v


def held(x, storage):
    if storage == 'bf16':
        return x.double()
    codes, scale = codes64(x, storage)
    return torch.from_numpy(codes * scale[..., None]).to(DEV)


@pytest.mark.parametrize('storage', STORAGES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('size, contexts', [
    (16, [1]), (16, [16, 0, 17, 15]), (64, [63, 200, 1, 65]),
    (256, [257, 3])])
def test_rows_read_back_as_their_codes(storage, dim, size, contexts):
    heads = 3
    cache, table, pack, k, v = filled(storage, contexts, size, heads, dim, 5)
    got_k, got_v = cache.read(table, pack)
    assert torch.equal(got_k, held(k, storage).to(torch.bfloat16))
    assert torch.equal(got_v, held(v, storage).to(torch.bfloat16))


@pytest.mark.parametrize('storage', ['int8', 'e4m3'])
def test_codes_of_ties_extremes_and_zeros(storage):
    dim = 64
    x = torch.zeros(9, 1, dim)
    x[0, 0] = torch.arange(dim) - 31.5  # ties of int8 around top = 32
    x[0, 0, 0] = 63.5 * 2
    x[1] = 0
    x[2, 0, 3] = 3e38
    x[2, 0, 4] = 1e36
    x[3, 0, 3] = 1e-30
    x[4, 0, 5] = 448.0
    x[4, 0, 6] = 1.0625  # a tie of e4m3
    x[4, 0, 7] = 1.1875
    x[5, 0, 5] = 449.0
    x[6, 0, :] = 2.0 ** torch.arange(-40, 24).float()
    x[7, 0, 1] = math.inf
    x[8, 0, 2] = math.nan
    x = x.to(torch.bfloat16).to(DEV)
    cache = kvcache.PagedCache.empty(1, 16, 1, dim, storage, DEV)
    poison(cache)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    pack = sequences.SequencePack([9], device=DEV)
    cache.write(x, -x, table, start, pack)
    codes, scale = codes64(x[:7], storage)
    assert np.array_equal(cache.k[0, 0, :7].float().cpu().numpy(),
                          codes[:, 0])
    assert np.array_equal(cache.k_scale[0, 0, :7].double().cpu().numpy(),
                          scale[:, 0])
    assert np.array_equal(cache.v[0, 0, :7].float().cpu().numpy(),
                          -codes[:, 0])
    assert cache.k_scale[0, 0, 7:9].isnan().all()
    k, _ = cache.read(table, pack)
    assert k[7:].isnan().all() and not k[:7].isnan().any()


@pytest.mark.parametrize('storage', STORAGES)
def test_write_touches_its_rows_only(storage):
    contexts, size, heads, dim = [40, 21], 16, 2, 64
    cache, table, pack, k, v = filled(storage, contexts, size, heads, dim, 9)
    before = [t.clone() for t in (cache.k.view(torch.uint8),
                                  cache.v.view(torch.uint8))]
    new = sequences.SequencePack([5, 3], device=DEV)
    starts = torch.tensor([14, 18], dtype=torch.int32, device=DEV)
    k2, v2 = rows(8, heads, dim, 31), rows(8, heads, dim, 32)
    cache.write(k2, v2, table, starts, new)
    want_k, want_v = k.clone(), v.clone()
    for want, got in ((want_k, k2), (want_v, v2)):
        want[14:19] = got[:5]
        want[40 + 18:40 + 21] = got[5:]
    got_k, got_v = cache.read(table, pack)
    assert torch.equal(got_k, held(want_k, storage).to(torch.bfloat16))
    assert torch.equal(got_v, held(want_v, storage).to(torch.bfloat16))
    kept = torch.ones(cache.k.shape[:3], dtype=torch.bool, device=DEV)
    for b, (s, n) in enumerate([(14, 5), (18, 3)]):
        for j in range(s, s + n):
            kept[table[b, j // size].long(), :, j % size] = False
    for old, now in zip(before, (cache.k, cache.v)):
        assert torch.equal(old[kept], now.view(torch.uint8)[kept])


def test_strided_rows_are_written():
    heads, dim = 2, 128
    cache = kvcache.PagedCache.empty(4, 16, heads, dim, 'bf16', DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    pack = sequences.SequencePack([20], device=DEV)
    fused = rows(20, 3 * heads, dim, 3)  # q, k, v of one projection
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    cache.write(k, v, table, start, pack)
    got = cache.read(table, pack)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    odd = rows(20, heads, dim + 1, 4)[:, :, 1:]  # no 16-byte pieces
    one = rows(20, 1, dim, 5).expand(20, heads, dim)
    cache.write(odd, one, table, start, pack)
    got = cache.read(table, pack)
    assert torch.equal(got[0], odd) and torch.equal(got[1], one)


def check_attend(cache, table, q, k, v, contexts, storage, scale=None):
    lengths = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q, table, lengths, scale, return_lse=True)
    n, heads, dim = q.shape
    kv_heads = cache.kv_heads
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    k, v = held(k, storage), held(v, storage)
    at = 0
    w = (2.0 ** -8 if storage == 'bf16' else 2.0 ** -11) + 2.0 ** -14
    for b, c in enumerate(contexts):
        kb, vb = k[at:at + c], v[at:at + c]
        at += c
        if c == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        kb, vb = (x.repeat_interleave(group, 1) for x in (kb, vb))
        qb = q[b].double()
        s = torch.einsum('hd,jhd->hj', qb, kb) * scale
        want_lse = torch.logsumexp(s, -1)
        p = torch.exp(s - want_lse[:, None])
        want = torch.einsum('hj,jhd->hd', p, vb)
        size = torch.einsum('hd,jhd->hj', qb.abs(), kb.abs()).amax(-1) * scale
        off = 2.0 ** -24 * (dim + 8) * size
        bound = ((w + 2 * off)[:, None] *
                 torch.einsum('hj,jhd->hd', p, vb.abs()) +
                 2.0 ** -8 * want.abs() + 1e-30)
        err = (out[b].double() - want).abs()
        assert (err <= bound).all(), (b, c, float((err / bound).max()))
        lse_bound = off + 2.0 ** -20 * (1 + want_lse.abs())
        err = (lse[b].double() - want_lse).abs()
        assert (err <= lse_bound).all(), (b, c, float((err / lse_bound).max()))
    return out


@pytest.mark.parametrize('storage', STORAGES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('size, contexts, heads, kv_heads', [
    (16, [1], 1, 1),
    (16, [15, 0, 16, 17, 1], 8, 2),
    (64, [700, 63, 0, 129, 1000], 14, 2),
    (32, [2500], 32, 4),
    (128, [333, 90, 20], 20, 1),   # 20 heads: two tiles of one kv head
    (256, [5, 513], 64, 2)])
def test_attend_matches_the_definition(storage, dim, size, contexts, heads,
                                       kv_heads):
    cache, table, _, k, v = filled(storage, contexts, size, kv_heads, dim, 11)
    q = rows(len(contexts), heads, dim, 77)
    check_attend(cache, table, q, k, v, contexts, storage)


@pytest.mark.parametrize('storage', STORAGES)
def test_attend_many_short_sequences(storage):
    # More sequences than a block's threads: every CTA has several pieces.
    contexts = [(7 * i) % 53 for i in range(300)]
    cache, table, _, k, v = filled(storage, contexts, 16, 2, 64, 13)
    q = rows(len(contexts), 6, 64, 78)
    check_attend(cache, table, q, k, v, contexts, storage)


@pytest.mark.parametrize('storage', STORAGES)
def test_attend_long_context_and_extreme_values(storage):
    contexts = [40000, 3]
    size, heads, dim = 64, 1, 128
    cache, table, pack, k, v = filled(storage, contexts, size, heads, dim, 17)
    gen = torch.Generator().manual_seed(5)
    # Rows of very unequal size: scales, maxima and references all move.
    k = k * torch.exp(1.5 * torch.randn(k.shape[0], 1, 1, generator=gen)
                      ).to(DEV).to(torch.bfloat16)
    v = v * torch.exp(3 * torch.randn(k.shape[0], 1, 1, generator=gen)
                      ).to(DEV).to(torch.bfloat16)
    v[100:200] = 0
    starts = torch.zeros(2, dtype=torch.int32, device=DEV)
    cache.write(k, v, table, starts, pack)
    q = rows(2, 5, dim, 79, 4.0)
    q[1] = 0
    check_attend(cache, table, q, k, v, contexts, storage)
    check_attend(cache, table, q * 2.0 ** -30, k, v, contexts, storage, 0.3)


@pytest.mark.parametrize('storage', STORAGES)
def test_attend_repeats_bit_for_bit_and_follows_the_lengths_in_a_graph(
        storage):
    contexts = [900, 64, 300]
    cache, table, _, k, v = filled(storage, contexts, 16, 2, 128, 19)
    q = rows(3, 8, 128, 80)
    lengths = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    first = cache.attend(q, table, lengths)
    assert torch.equal(first, cache.attend(q, table, lengths))
    shorter = torch.tensor([17, 0, 299], dtype=torch.int32, device=DEV)
    want = cache.attend(q, table, shorter)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    with torch.cuda.stream(side):
        for g in graphs:
            with torch.cuda.graph(g, stream=side):
                outs.append(cache.attend(q, table, lengths))
    for g, out in zip(graphs, outs):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    lengths.copy_(shorter)
    for g, out in zip(graphs, outs):
        g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)


def test_offsets_past_32_bits():
    # Rows of the last pages lie more than 2^32 bytes into the tensors.
    size, heads, dim = 256, 8, 128
    n_pages = 9000  # 9000 * 8 * 256 * 256 bytes = 4.7 GB each
    cache = kvcache.PagedCache.empty(n_pages, size, heads, dim, 'bf16', DEV)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32,
                         device=DEV)
    contexts = [2 * size + 40]
    pack = sequences.SequencePack(contexts, device=DEV)
    k, v = (rows(contexts[0], heads, dim, s) for s in (1, 2))
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.write(k, v, table, start, pack)
    got = cache.read(table, pack)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    check_attend(cache, table, rows(1, 16, dim, 3), k, v, contexts, 'bf16')


@pytest.mark.parametrize('storage', STORAGES)
def test_places_that_do_not_exist_are_reported_and_touch_nothing(storage):
    size, heads, dim = 16, 2, 64
    cache, table, pack, k, v = filled(storage, [20, 20], size, heads, dim, 23)
    before = cache.k.view(torch.uint8).clone()
    start = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (-1, cache.n_pages, 2 ** 31 - 1):
        t = table.clone()
        t[0, 1] = bad
        cache.write(k, v, t, start, pack)
        assert _lib.device_status(reset=True) == _lib.VEDA_ERR_INVALID
        assert torch.equal(before, cache.k.view(torch.uint8))
        got, _ = cache.read(t, pack)
        assert _lib.device_status(reset=True) == _lib.VEDA_ERR_INVALID
        assert (got[16:20] == 0).all()
        assert torch.equal(got[20:], held(k[20:], storage).bfloat16())
        lengths = torch.tensor([20, 20], dtype=torch.int32, device=DEV)
        out = cache.attend(rows(2, 2, dim, 3), t, lengths)
        assert _lib.device_status(reset=True) == _lib.VEDA_ERR_INVALID
        assert out.isfinite().all()
    for starts in ([-1, 0], [13, 0], [2 ** 31 - 8, 0]):
        t = torch.tensor(starts, dtype=torch.int32, device=DEV)
        cache.write(k, v, table, t, pack)
        assert _lib.device_status(reset=True) == _lib.VEDA_ERR_INVALID
        cache.write(k, v, table, start, pack)
        got, _ = cache.read(table, pack)
        assert torch.equal(got, held(k, storage).bfloat16())
    for n in (-5, 33, 2 ** 31 - 1):
        lengths = torch.tensor([20, n], dtype=torch.int32, device=DEV)
        cache.attend(rows(2, 2, dim, 3), table, lengths)
        assert _lib.device_status(reset=True) == _lib.VEDA_ERR_INVALID


@pytest.mark.parametrize('storage', STORAGES)
def test_a_wider_table_and_shared_pages(storage):
    # A slice of a wider table, and two sequences that read one prefix page.
    contexts, size, dim = [40, 33], 16, 64
    cache, table, _, k, v = filled(storage, contexts, size, 2, dim, 37)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=DEV)
    wide[:, :3] = table
    wide[1, 0] = wide[0, 0]
    k, v = k.clone(), v.clone()
    for t in (k, v):
        t[40:56] = t[:16]
    got, _ = cache.read(wide[:, :3], sequences.SequencePack(contexts,
                                                            device=DEV))
    assert torch.equal(got, held(k, storage).bfloat16())
    q = rows(2, 4, dim, 5)
    check_attend(cache, wide[:, :3], q, k, v, contexts, storage)
    check_attend(cache, wide, q, k, v, contexts, storage)


def test_many_heads_share_a_key_head():
    contexts = [70, 9]
    cache, table, _, k, v = filled('int8', contexts, 16, 1, 128, 41)
    check_attend(cache, table, rows(2, 130, 128, 6), k, v, contexts, 'int8')


def test_no_rows_and_other_streams():
    cache, table, pack, k, v = filled('int8', [30, 5], 16, 2, 64, 29)
    none = sequences.SequencePack([0, 0], device=DEV)
    start = torch.zeros(2, dtype=torch.int32, device=DEV)
    cache.write(k[:0], v[:0], table, start, none)
    got = cache.read(table, none)
    assert got[0].shape == (0, 2, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.read(table, sequences.SequencePack([30, 5], device=DEV))
    side.synchronize()
    assert torch.equal(got[0], held(k, 'int8').bfloat16())


def test_calls_on_two_streams():
    contexts = [3000, 0, 500]
    cache, table, _, k, v = filled('e4m3', contexts, 64, 2, 128, 43)
    q = rows(3, 8, 128, 7)
    lengths = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    want = cache.attend(q, table, lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for s, out in zip(streams, outs):
            with torch.cuda.stream(s):
                out.append(cache.attend(q, table, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for out in outs for o in out)


@pytest.mark.parametrize('storage', STORAGES)
@pytest.mark.parametrize('dim', [64, 128])
def test_sums_over_long_runs_of_keys_do_not_drift(storage, dim):
    """Many contexts (here of shared pages) make a warp's run of keys long, and
    equal weights make the result small beside the values: the mean of n
    values, whose sums may lose fp32's bits only of what they add up."""
    n, rows_, heads = 512, 32768, 2
    gen = torch.Generator().manual_seed(61)
    # Integers with the same largest magnitude in every row: every weight times
    # its scale is the same power of two, and no weight is rounded.
    v = torch.randint(-14, 15, (rows_, heads, dim), generator=gen).float() * 8
    v[:, :, 3] = 127
    v = v.bfloat16().to(DEV)
    k = rows(rows_, heads, dim, 62)
    cache = kvcache.PagedCache.empty(rows_ // 256, 256, heads, dim, storage,
                                     DEV)
    table = torch.arange(rows_ // 256, dtype=torch.int32, device=DEV)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    pack = sequences.SequencePack([rows_], device=DEV)
    cache.write(k, v, table[None], start, pack)
    q = torch.zeros(n, 4, dim, dtype=torch.bfloat16, device=DEV)
    out = cache.attend(q, table.repeat(n, 1),
                       torch.full((n,), rows_, dtype=torch.int32, device=DEV))
    want = held(v, storage).mean(0).repeat_interleave(2, 0)
    size = held(v, storage).abs().mean(0).repeat_interleave(2, 0)
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -14 * size
    assert ((out.double() - want).abs() <= bound).all()


def defined(q, k, v, scale, w):
    """(out, lse) of one sequence's query [heads, D] over the rows k, v
    [n, kv_heads, D] (fp64, as held), and their bounds (see above)."""
    group = q.shape[0] // k.shape[1]
    k, v = (x.repeat_interleave(group, 1) for x in (k, v))
    q = q.double()
    s = torch.einsum('hd,jhd->hj', q, k) * scale
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    want = torch.einsum('hj,jhd->hd', p, v)
    size = torch.einsum('hd,jhd->hj', q.abs(), k.abs()).amax(-1) * scale
    off = 2.0 ** -24 * (q.shape[1] + 8) * size
    bound = ((w + 2.0 ** -14 + 2 * off)[:, None] *
             torch.einsum('hj,jhd->hd', p, v.abs()) +
             2.0 ** -8 * want.abs() + 1e-30)
    return want, bound, lse, off + 2.0 ** -20 * (1 + lse.abs())


@pytest.mark.parametrize('storage', STORAGES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('heads', [2, 40])
def test_keys_of_pages_that_do_not_exist_are_absent(storage, dim, heads):
    """The attention is that over the other keys, whichever page of a context
    is missing; without any it is that of a context without rows."""
    size = 16
    contexts = [20, 40, 70, 33, 3000, 3000]
    missing = [{1}, {0}, {1, 2}, {0, 1, 2}, set(range(1, 188, 3)),
               set(range(188))]
    cache, table, _, k, v = filled(storage, contexts, size, 2, dim, 47)
    bad = [-1, cache.n_pages, 2 ** 31 - 1]
    for b, pages in enumerate(missing):
        for i, page in enumerate(pages):
            table[b, page] = bad[(b + i) % 3]
    q = rows(len(contexts), heads, dim, 48)
    lengths = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q, table, lengths, return_lse=True)
    assert _lib.device_status(reset=True) == _lib.VEDA_ERR_INVALID
    k, v = held(k, storage), held(v, storage)
    w = 2.0 ** -8 if storage == 'bf16' else 2.0 ** -11
    at = 0
    for b, c in enumerate(contexts):
        keep = torch.tensor([j // size not in missing[b] for j in range(c)],
                            device=DEV)
        kb, vb = k[at:at + c][keep], v[at:at + c][keep]
        at += c
        if not keep.any():
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        want, bound, want_lse, lse_bound = defined(q[b], kb, vb, dim ** -0.5,
                                                   w)
        assert ((out[b].double() - want).abs() <= bound).all(), b
        assert ((lse[b].double() - want_lse).abs() <= lse_bound).all(), b


@pytest.mark.parametrize('storage', STORAGES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('place', [0, 5, 150, 2999])
@pytest.mark.parametrize('power', [20, 30, 60])
def test_a_large_value_row_without_weight_costs_no_bits(storage, dim, place,
                                                        power):
    """A value row that nothing attends to may be any number of times larger
    than those that are attended to."""
    contexts, heads = [3000, 40], 3
    cache, table, pack, k, v = filled(storage, contexts, 64, heads, dim, 51)
    q = rows(2, heads, dim, 52)
    # Its score is about -16 |q|^2 scale: -128 at least.
    k[place], v[place] = -16 * q[0], v[place] * 2.0 ** power
    starts = torch.zeros(2, dtype=torch.int32, device=DEV)
    cache.write(k, v, table, starts, pack)
    check_attend(cache, table, q, k, v, contexts, storage)


@pytest.mark.parametrize('storage', STORAGES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('place', [0, 77])
def test_a_row_with_all_the_weight_may_hold_the_smallest_values(storage, dim,
                                                                place):
    """A key that takes nearly all the weight and has values of 2^-40 leaves
    the others' their bits: weights of e^-20 and values of 1."""
    contexts, heads = [400], 2
    cache, table, pack, k, v = filled(storage, contexts, 16, heads, dim, 53)
    q = rows(1, heads, dim, 54)
    scale = dim ** -0.5
    top = q[0].double().square().sum(-1, keepdim=True) * scale
    k = (k * 0.05).bfloat16()
    k[place] = (q[0].double() * (20 / top)).bfloat16()
    v[place] = (v[place] * 2.0 ** -40).bfloat16()
    starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.write(k, v, table, starts, pack)
    check_attend(cache, table, q, k, v, contexts, storage)


def pages_of(cache):
    return [t.clone().view(torch.uint8) for t in
            (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


@pytest.mark.parametrize('storage', STORAGES)
def test_rows_of_no_sequence_are_left_as_they_are(storage):
    """Offsets on the device that begin behind the first row or end before the
    last (a padded batch): the rows outside are neither stored nor read."""
    size, heads, dim = 16, 2, 64
    cache, table, pack, k, v = filled(storage, [40, 48], size, heads, dim, 57)
    starts = torch.tensor([3, 30], dtype=torch.int32, device=DEV)
    new_k, new_v = rows(20, heads, dim, 58), rows(20, heads, dim, 59)
    offsets = torch.tensor([4, 9, 15], dtype=torch.int32, device=DEV)
    exact = sequences.SequencePack([5, 6], device=DEV)
    cache.write(new_k[4:15], new_v[4:15], table, starts, exact)
    want = pages_of(cache)
    cache.write(k, v, table, torch.zeros_like(starts), pack)
    padded = sequences.SequencePack([10, 10], device=DEV)
    padded.q_offsets.copy_(offsets)
    cache.write(new_k, new_v, table, starts, padded)
    assert all(torch.equal(a, b) for a, b in zip(want, pages_of(cache)))
    got = [torch.full((20, heads, dim), 7.0, dtype=torch.bfloat16, device=DEV)
           for _ in range(2)]
    short = cache.read(table, exact)
    _lib.call_on(0, 'veda_cache_read', *cache._view(table, 2),
                 offsets.data_ptr(), 20, *(t.data_ptr() for t in got))
    for t, inside in zip(got, short):
        assert torch.equal(t[4:15], inside)
        assert (t[:4] == 7).all() and (t[15:] == 7).all()
