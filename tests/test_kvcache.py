"""The paged cache and packed sequences on the host: refusals, and the work
tables against a walk over every (query, key) pair. No GPU needed."""

import numpy as np
import pytest
import torch

from miowtion_b200 import kvcache
from miowtion_b200 import sequences


def pack(q, k=None):
    return sequences.SequencePack(q, k, 'cpu')


def cache(storage='int8', pages=4, size=16, heads=2, dim=64):
    return kvcache.PagedCache.empty(pages, size, heads, dim, storage, 'cpu')


@pytest.mark.parametrize('lengths, match', [
    ([], 'non-empty'), ([1.5], 'integers'), ([3, -1], 'negative'),
    ([[1, 2]], 'non-empty'), ([2 ** 31], 'below'),
    ([2 ** 30, 2 ** 30], 'fewer than')])
def test_pack_refuses(lengths, match):
    with pytest.raises(ValueError, match=match):
        pack(lengths)


def test_pack_refuses_other_sequence_counts():
    with pytest.raises(ValueError, match='same'):
        pack([1, 2], [1, 2, 3])


def test_pack_properties():
    p = pack([3, 0, 5], [4, 7, 5])
    assert (p.total_q, p.total_k, p.n_sequences) == (8, 16, 3)
    assert p.q_offsets.tolist() == [0, 3, 3, 8]
    assert p.k_offsets.tolist() == [0, 4, 11, 16]
    assert not p.whole and not p.single_tokens
    with pytest.raises(ValueError):
        p.q_lengths[0] = 5
    assert pack([1, 1], [5, 1]).single_tokens and pack([2, 0]).whole


@pytest.mark.parametrize('group', [1, 3, 8, 128])
@pytest.mark.parametrize('q, k', [
    ([1], [1]), ([129, 0, 1], [129, 0, 1]), ([5, 300], [400, 301]),
    ([200, 7], [90, 0]), ([0, 0], [3, 0]), ([130], [513])])
def test_work_items_cover_every_visible_pair_once(group, q, k):
    forward, query, key, n_tiles = sequences.work_items(
        np.array(q), np.array(k), group)
    tokens = 128 // group
    p = pack(q, k)
    want = np.zeros((p.total_q, p.total_k), bool)
    q0, k0 = np.cumsum([0] + q), np.cumsum([0] + k)
    for b in range(len(q)):
        for i in range(q[b]):
            want[q0[b] + i, k0[b]:k0[b] + max(0, i + 1 + k[b] - q[b])] = True
    for items, per_item in ((forward, 2), (query, 1)):
        got = np.zeros_like(want)
        rows = np.zeros(p.total_q, int)
        for row, n, kr, kpos, c, blocks, tile, _ in items:
            assert 1 <= n <= per_item * tokens and 0 <= tile < n_tiles
            rows[row:row + n] += 1
            for t in range(n):
                seen = min(c, max(0, kpos + t + 1))
                assert seen <= 128 * blocks
                got[row + t, kr:kr + seen] = True
        assert (rows == 1).all() and np.array_equal(got, want)
        assert (np.diff(items[:, 5]) <= 0).all()
    got = np.zeros_like(want)
    keys = np.zeros(p.total_k, int)
    tiles = set()
    for row, n, qr, nq, shift, first, blocks, base in key:
        assert 1 <= n <= 128
        keys[row:row + n] += 1
        for blk in range(blocks):
            t0 = (first + blk) * tokens
            assert t0 < nq
            tiles.add(base + first + blk)
            for t in range(t0, min(nq, t0 + tokens)):
                seen = min(n, max(0, t - shift + 1))
                got[qr + t, row:row + seen] = True
    assert (keys == 1).all() and np.array_equal(got, want)
    assert tiles <= set(range(n_tiles))


@pytest.mark.parametrize('q, k, group, kv_heads, sms', [
    ([64] * 3, [9000, 8000, 300], 4, 2, 148), ([1], [100000], 8, 1, 148),
    ([1000, 40], [1000, 40], 1, 8, 148), ([500], [7000], 7, 2, 16),
    ([64, 64], [1, 1], 4, 2, 148)])
def test_split_items_are_the_whole_ones(q, k, group, kv_heads, sms):
    whole, _, _, _ = sequences.work_items(np.array(q), np.array(k), group)
    items, joins, n_parts = sequences.split_items(whole, kv_heads, sms)
    assert (np.diff(items[:, 5]) <= 0).all()
    parts = {}
    for it in items:
        parts.setdefault((it[0], it[1]), []).append(tuple(it[5:]))
    join_of = {(j[0], j[1]): (j[2], j[3]) for j in joins}
    assert len(parts) == len(whole)
    for it in whole:
        own = sorted(parts[it[0], it[1]], key=lambda x: x[1])
        at = 0
        for blocks, first, _ in own:
            assert first == at
            at += blocks
        assert at == it[5]
        if len(own) == 1:
            assert own[0][2] == -1 and (it[0], it[1]) not in join_of
        else:
            assert min(b for b, _, _ in own) >= 2
            start, count = join_of[it[0], it[1]]
            assert [x[2] for x in own] == list(range(start, start + count))
    numbers = [it[7] for it in items if it[7] >= 0]
    assert sorted(numbers) == list(range(n_parts))


def test_group_is_bounded():
    for group in (0, 129):
        with pytest.raises(ValueError, match='share'):
            sequences.work_items(np.array([4]), np.array([4]), group)


def test_cache_refuses_wrong_pages():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.zeros(4, 2, 16)
    good = dict(k=k, v=k, k_scale=s, v_scale=s)
    kvcache.PagedCache(**good)
    for change, match in [
            (dict(v=k[:3]), 'one shape'), (dict(k_scale=None), 'scales'),
            (dict(v_scale=s.double()), 'scales'),
            (dict(k_scale=s[:, :, :8]), 'scales'),
            (dict(k=k.float(), v=k.float()), 'pages are'),
            (dict(k=k.bfloat16(), v=k.bfloat16()), 'no scales'),
            (dict(k=k.transpose(0, 1), v=k.transpose(0, 1),
                  k_scale=s.transpose(0, 1), v_scale=s.transpose(0, 1)),
             'contiguous')]:
        with pytest.raises(ValueError, match=match):
            kvcache.PagedCache(**{**good, **change})
    for size, dim, match in [(8, 64, 'page_size'), (24, 64, 'page_size'),
                             (512, 64, 'page_size'), (16, 96, 'head dim')]:
        with pytest.raises(ValueError, match=match):
            cache(size=size, dim=dim)
    with pytest.raises(ValueError, match='storage'):
        cache('fp4')


def test_cache_calls_refuse_wrong_arguments():
    c = cache()
    p = pack([3, 2])
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 1, dtype=torch.int32)
    starts = torch.zeros(2, dtype=torch.int32)
    for args, match in [
            ((k[:4], k, table, starts, p), 'k must be'),
            ((k, k.float(), table, starts, p), 'v must be'),
            ((k, k, table.long(), starts, p), 'table must be'),
            ((k, k, table[:1], starts, p), 'table must be'),
            ((k, k, table[:, :0], starts, p), 'one page'),
            ((k, k, table, starts[:1], p), 'starts must be')]:
        with pytest.raises(ValueError, match=match):
            c.write(*args)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    for args, match in [
            ((q[:, :3], table, starts), 'multiple'),
            ((q[:, :, :32], table, starts), 'q must be'),
            ((q.float(), table, starts), 'q must be'),
            ((q, table, starts.float()), 'lengths must be'),
            ((q, table, starts, 0.0), 'scale'),
            ((q, table, starts, float('nan')), 'scale'),
            ((q.clone().requires_grad_(), table, starts), 'no gradient')]:
        with pytest.raises(ValueError, match=match):
            c.attend(*args)
    with pytest.raises(ValueError, match='table must be'):
        c.read(table[:1], p)


def test_the_pages_of_a_cache_are_fixed():
    c = cache()
    with pytest.raises(AttributeError):
        c.k = c.v


def test_cache_calls_refuse_to_fall_back():
    c = cache('bf16')
    p = pack([1])
    k = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(1, 1, dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: c.write(k, k, table, one, p),
                 lambda: c.read(table, p), lambda: c.attend(k, table, one)):
        with pytest.raises(NotImplementedError, match='unavailable'):
            call()


def test_causal_attention_refuses():
    from miowtion_b200 import kernels
    p = pack([3, 2])
    q = torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    for args, match in [
            ((q, k, k[:4], p), 'one shape'), ((q[0], k, k, p), 'rows, heads'),
            ((q[:, :, :32], k[:, :, :32], k[:, :, :32], p), 'head dim'),
            ((q, k[:, :, :32], k[:, :, :32], p), 'head dim'),
            ((q[:, :3], k, k, p), 'key heads'),
            ((q[:4], k, k, p), 'rows, not'), ((q, k[:4], k[:4], p), 'rows, not'),
            ((q.half(), k, k, p), 'bf16'), ((q, k, k, p, -1.0), 'scale'),
            ((q, k, k, p, float('inf')), 'scale')]:
        with pytest.raises(ValueError, match=match):
            kernels.causal_attention(*args)
    wide = torch.zeros(5, 130, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='1 to 128'):
        kernels.causal_attention(wide, k[:, :1], k[:, :1], p)
    with pytest.raises(NotImplementedError, match='unavailable'):
        kernels.causal_attention(q, k, k, p)


@pytest.mark.parametrize('scale', [0.0, 1e-40, 1e38, 1e300, float('nan')])
def test_scales_that_fp32_does_not_hold_are_refused(scale):
    from miowtion_b200 import kernels
    with pytest.raises(ValueError, match='positive and finite'):
        kernels.softmax_scale(scale, 64)


@pytest.mark.parametrize('lengths, kv_heads, sms', [
    ([8192, 5000, 1000], 4, 148), ([700, 9, 0, 130], 3, 7), ([1], 1, 4),
    ([500] * 40, 2, 148), ([300, 200], 1, 5), ([4096], 2, 5)])
def test_deal_takes_every_key_item_once(lengths, kv_heads, sms):
    lengths = np.array(lengths, np.int64)
    _, _, key, _ = sequences.work_items(lengths, lengths, 4)
    blocks = key[:, 6]
    turns = sequences.deal_items(blocks, kv_heads, sms)
    items = len(key) * kv_heads
    if not sms < items <= sequences.MOST_TURNS * sms:
        assert turns.shape == (0, sms)
        return
    assert turns.shape[1] == sms
    assert sorted(turns[turns >= 0]) == list(range(items))
    # A processor's turns end once.
    assert ((turns[1:] < 0) | (turns[:-1] >= 0)).all()
    cost = np.append(np.repeat(blocks + sequences.ITEM_COST, kv_heads), 0.0)
    load = cost[turns].sum(0)
    # Each item went to one of the half that had least: twice the mean at most.
    assert load.max() <= 2 * cost.sum() / sms + cost.max()


def test_forward_mode_derivatives_are_refused():
    """A dual tensor has no requires_grad, and a kernel would read its values
    and drop its tangent."""
    from torch.autograd import forward_ad

    from miowtion_b200 import kernels
    p = pack([3, 2])
    q = torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    c = cache('bf16')
    table = torch.zeros(2, 1, dtype=torch.int32)
    two = torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros(128, 2, 128, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: kernels.causal_attention(dual(q), k, k, p),
                 lambda: kernels.causal_attention(q, dual(k), k, p),
                 lambda: kernels.causal_attention(q, k, dual(k), p),
                 lambda: c.write(dual(k), k, table, two, p),
                 lambda: c.write(k, dual(k), table, two, p),
                 lambda: c.attend(dual(q[:2]), table, two),
                 lambda: kernels.block_sparse_attention(
                     rows, rows, dual(rows), None, None)]
        for call in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad):
                    with pytest.raises(ValueError, match='forward-mode'):
                        call()
        # Without tangents, or where they are switched off, as ever.
        with pytest.raises(NotImplementedError, match='unavailable'):
            kernels.causal_attention(q, k, k, p)
        with torch.inference_mode():
            with pytest.raises(NotImplementedError, match='unavailable'):
                kernels.causal_attention(dual(q), k, k, p)


def test_a_write_refuses_rows_whose_gradient_it_would_lose():
    c = cache('bf16')
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    leaf = k.clone().requires_grad_()
    table = torch.zeros(2, 1, dtype=torch.int32)
    two = torch.zeros(2, dtype=torch.int32)
    for args in ((leaf, k), (k, leaf), (leaf * 2, k)):
        with pytest.raises(ValueError, match='no gradient'):
            c.write(*args, table, two, pack([1, 1]))
        with torch.no_grad():
            with pytest.raises(NotImplementedError, match='unavailable'):
                c.write(*args, table, two, pack([1, 1]))


@pytest.mark.parametrize('shape', [(), (64,), (5, 64), (5, 4, 0), (1, 5, 4, 64)])
def test_causal_attention_refuses_other_ranks_and_empty_heads(shape):
    from miowtion_b200 import kernels
    q = torch.zeros(shape, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='rows, heads|head dim'):
        kernels.causal_attention(q, q, q, pack([3, 2]))
