"""Causal attention of packed sequences against its definition in 64 bits.

Bounds count the roundings of the forward: weights to bf16 (half a step,
2^-8, relative), the output to bf16 (2^-8) and what the fp32 scores are off,
    |out - want| <= (2^-8 + 2 s + 2^-14) sum_j p_j |v_j| + 2^-8 |want|
with s = (D + 8) 2^-24 A for scores of total size A = scale max_j sum_d
|q_d k_jd| (a relative error of a weight, and again of the weights' sum).

Gradients: with half steps u = 2^-8 of P, dS and the stored gradient, of the
stored out in D = rowsum(dO O), and e = 2 s + 2^-14 relative in P,
    |dv_j - want| <= (u + e) sum_i p_ij |do_i| + u |want|,
    |ds_ij - want| <= (u + e) |ds_ij| + p_ij u sum_d |do_id out_id|
                      + p_ij 2^-16 sum_d |do_id| (|v_jd| + |out_id|),
and dq, dk bounded by scale times the sums of these against |k| and |q|, plus
u |want|.
"""

import math

import pytest
import torch

from miowtion_b200 import _lib
from miowtion_b200 import kernels
from miowtion_b200 import sequences

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.device_status(reset=True)
    yield
    assert _lib.device_status(reset=True) == 0, 'the status word was set'


def rows(n, heads, dim, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=gen) * scale
    return x.to(torch.bfloat16).to(DEV)


def problem(q_lengths, k_lengths, heads, kv_heads, dim, seed=3, scale=1.0):
    pack = sequences.SequencePack(q_lengths, k_lengths, DEV)
    q = rows(pack.total_q, heads, dim, seed, scale)
    k, v = (rows(pack.total_k, kv_heads, dim, seed + i) for i in (1, 2))
    return pack, q, k, v


def each_head(pack, q, k):
    """(query rows, key rows, query head, key head, mask) of every pair."""
    group = q.shape[1] // k.shape[1]
    i0 = j0 = 0
    for n, c in zip(pack.q_lengths.tolist(), pack.k_lengths.tolist()):
        i = torch.arange(n, device=DEV)[:, None]
        j = torch.arange(c, device=DEV)[None, :]
        for h in range(q.shape[1]):
            yield (slice(i0, i0 + n), slice(j0, j0 + c), h, h // group,
                   j <= i + c - n)
        i0, j0 = i0 + n, j0 + c


def softmax64(q, k, sees, scale):
    s = (scale * q @ k.T).masked_fill(~sees, -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[1] else torch.full(
        s.shape[:1], -math.inf, device=DEV, dtype=torch.float64)
    p = torch.exp(s - lse[:, None]).masked_fill(~sees, 0.0)
    return p, lse


def check_forward(pack, q, k, v, out, lse, scale=None):
    dim = q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    assert out.isfinite().all()
    for at, keys, h, hk, sees in each_head(pack, q, k):
        qb, kb, vb = q[at, h].double(), k[keys, hk].double(), v[
            keys, hk].double()
        p, want_lse = softmax64(qb, kb, sees, scale)
        want = p @ vb
        if kb.shape[0] == 0 or qb.shape[0] == 0:
            assert (out[at, h] == 0).all()
            continue
        size = ((qb.abs() @ kb.abs().T) * sees).amax(-1) * scale
        off = 2.0 ** -24 * (dim + 8) * size
        bound = ((2.0 ** -8 + 2.0 ** -14 + 2 * off)[:, None] * (
            p @ vb.abs()) + 2.0 ** -8 * want.abs() + 1e-30)
        err = (out[at, h].double() - want).abs()
        assert (err <= bound).all(), (h, float((err / bound).max()))
        empty = want_lse == -math.inf
        assert torch.equal(lse[at, h] == -math.inf, empty)
        err = (lse[at, h].double() - want_lse).abs()[~empty]
        bound = (off + 2.0 ** -20 * (1 + want_lse.abs()))[~empty]
        assert (err <= bound).all(), (h, float((err / bound).max()))


SHAPES = [
    # q lengths, k lengths, heads, key heads
    ([1], None, 1, 1),
    ([128], None, 2, 2),
    ([129, 1, 127], None, 3, 3),
    ([300, 0, 17, 64], None, 4, 1),
    ([5, 260], [400, 261], 6, 2),        # groups of 3: 126 rows of a tile
    ([200, 7, 30], [90, 0, 300], 8, 1),  # rows without a key
    ([1, 1, 1], [513, 1, 77], 14, 2),    # single tokens, groups of 7
    ([37, 90], None, 128, 1),            # a token fills a tile
    ([40], [170], 100, 1),
    ([700, 650], None, 16, 2),
]


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('q_lengths, k_lengths, heads, kv_heads', SHAPES)
def test_forward_matches_the_definition(q_lengths, k_lengths, heads, kv_heads,
                                        dim):
    pack, q, k, v = problem(q_lengths, k_lengths, heads, kv_heads, dim)
    out, lse = kernels.causal_attention(q, k, v, pack, return_lse=True)
    check_forward(pack, q, k, v, out, lse)


@pytest.mark.parametrize('dim', [64, 128])
def test_forward_of_more_items_than_processors(dim):
    lengths = [(37 * i) % 211 for i in range(90)]
    pack, q, k, v = problem(lengths, None, 8, 4, dim)
    out, lse = kernels.causal_attention(q, k, v, pack, return_lse=True)
    check_forward(pack, q, k, v, out, lse)


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('q_lengths, k_lengths, heads, kv_heads', [
    ([70, 5], [6000, 3001], 8, 2), ([1], [20000], 14, 2),
    ([33, 300, 9], [4000, 300, 0], 6, 2)])
def test_forward_of_items_cut_along_the_keys(q_lengths, k_lengths, heads,
                                             kv_heads, dim):
    pack, q, k, v = problem(q_lengths, k_lengths, heads, kv_heads, dim)
    assert pack.tables(heads // kv_heads, kv_heads).n_parts > 0
    out, lse = kernels.causal_attention(q, k, v, pack, return_lse=True)
    check_forward(pack, q, k, v, out, lse)
    dout = rows(pack.total_q, heads, dim, 9)
    check_gradients(pack, q, k, v, dout, gradients(pack, q, k, v, dout))


def test_forward_of_scores_that_grow_along_the_keys():
    # Maxima rise from tile to tile, so the accumulator is rescaled, and a
    # scale of its own.
    pack, q, k, v = problem([1000], None, 4, 2, 128)
    ramp = torch.linspace(0.05, 6.0, 1000, device=DEV)[:, None, None]
    k = (k.abs() * ramp).to(torch.bfloat16)
    q = q.abs()
    out, lse = kernels.causal_attention(q, k, v, pack, 0.05, return_lse=True)
    check_forward(pack, q, k, v, out, lse, 0.05)


def test_forward_of_strided_and_broadcast_inputs():
    pack, _, _, _ = problem([200, 90], None, 4, 2, 64)
    fused = rows(290, 8, 64, 5)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    out, lse = kernels.causal_attention(q, k, v, pack, return_lse=True)
    check_forward(pack, q, k, v, out, lse)
    k = rows(290, 1, 64, 6).expand(290, 2, 64)
    v = rows(290, 2, 65, 7)[:, :, 1:]
    out, lse = kernels.causal_attention(q, k, v, pack, return_lse=True)
    check_forward(pack, q, k, v, out, lse)


@pytest.mark.parametrize('dim', [64, 128])
def test_sequences_do_not_reach_one_another(dim):
    pack, q, k, v = problem([150, 70, 33], [150, 200, 33], 6, 2, dim)
    want, want_lse = kernels.causal_attention(q, k, v, pack, return_lse=True)
    q[150:220] = math.nan
    k[150:350] = math.inf
    v[150:350] = math.nan
    out, lse = kernels.causal_attention(q, k, v, pack, return_lse=True)
    for got, ref in ((out, want), (lse, want_lse)):
        assert torch.equal(got[:150], ref[:150])
        assert torch.equal(got[220:], ref[220:])
    assert out[150:220].isnan().all()


def gradients(pack, q, k, v, dout, scale=None):
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    out = kernels.causal_attention(*leaves, pack, scale)
    return torch.autograd.grad(out, leaves, dout)


def check_gradients(pack, q, k, v, dout, grads, scale=None):
    dim = q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    want = [torch.zeros(t.shape, dtype=torch.float64, device=DEV)
            for t in (q, k, v)]
    bound = [torch.zeros_like(t) for t in want]
    u = 2.0 ** -8
    for at, keys, h, hk, sees in each_head(pack, q, k):
        qb, kb, vb = q[at, h].double(), k[keys, hk].double(), v[
            keys, hk].double()
        if 0 in (qb.shape[0], kb.shape[0]):
            continue
        g = dout[at, h].double()
        p, _ = softmax64(qb, kb, sees, scale)
        out = p @ vb
        size = ((qb.abs() @ kb.abs().T) * sees).amax(-1) * scale
        e = 2 * 2.0 ** -24 * (dim + 8) * size[:, None] + 2.0 ** -14
        ds = p * (g @ vb.T - (g * out).sum(-1, keepdim=True))
        off = ((u + e) * ds.abs() +
               p * u * (g * out).abs().sum(-1, keepdim=True) +
               p * 2.0 ** -16 * (g.abs() @ vb.abs().T +
                                 (g * out).abs().sum(-1, keepdim=True)))
        want[0][at, h] += scale * ds @ kb
        want[1][keys, hk] += scale * ds.T @ qb
        want[2][keys, hk] += p.T @ g
        bound[0][at, h] += scale * off @ kb.abs()
        bound[1][keys, hk] += scale * off.T @ qb.abs()
        bound[2][keys, hk] += ((u + e) * p).T @ g.abs()
    for name, got, ref, off in zip(('dq', 'dk', 'dv'), grads, want, bound):
        assert got.isfinite().all(), name
        err = (got.double() - ref).abs()
        off = off + u * ref.abs() + 1e-30
        assert (err <= off).all(), (name, float((err / off).max()))


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('q_lengths, k_lengths, heads, kv_heads', SHAPES)
def test_gradients_match_the_definition(q_lengths, k_lengths, heads, kv_heads,
                                        dim):
    pack, q, k, v = problem(q_lengths, k_lengths, heads, kv_heads, dim)
    dout = rows(pack.total_q, heads, dim, 9)
    grads = gradients(pack, q, k, v, dout)
    check_gradients(pack, q, k, v, dout, grads)
    again = gradients(pack, q, k, v, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize('dim', [64, 128])
def test_gradients_of_more_items_than_processors(dim):
    lengths = [(37 * i) % 211 for i in range(90)]
    pack, q, k, v = problem(lengths, None, 8, 4, dim)
    dout = rows(pack.total_q, 8, dim, 9)
    check_gradients(pack, q, k, v, dout, gradients(pack, q, k, v, dout))


def test_gradients_agree_with_differences():
    pack, q, k, v = problem([60, 150], [90, 150], 4, 2, 64)
    dout = rows(pack.total_q, 4, 64, 9)
    grads = gradients(pack, q, k, v, dout)

    def loss(*args):
        total = 0.0
        for at, keys, h, hk, sees in each_head(pack, args[0], args[1]):
            p, _ = softmax64(args[0][at, h], args[1][keys, hk], sees, 0.125)
            total = total + (p @ args[2][keys, hk] *
                             dout[at, h].double()).sum()
        return float(total)

    base = [t.double() for t in (q, k, v)]
    for n, grad in enumerate(grads):
        way = rows(*base[n].shape, 40 + n).double()
        step = 1e-4
        plus, minus = ([t + s * way if m == n else t
                        for m, t in enumerate(base)] for s in (step, -step))
        slope = (loss(*plus) - loss(*minus)) / (2 * step)
        # Each gradient is off by at most a few 2^-8 of its size, with
        # independent signs along the direction: far below the sum of sizes.
        size = float((grad.double() * way).abs().sum())
        got = float((grad.double() * way).sum())
        assert abs(got - slope) <= 2.0 ** -8 * size, (n, got, slope)


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('q_lengths, k_lengths, heads, kv_heads', [
    ([300, 1, 70], None, 4, 2), ([70, 5], [6000, 3001], 8, 2),
    ([40, 200], [90, 30], 3, 1)])
def test_out_and_its_low_bits(q_lengths, k_lengths, heads, kv_heads, dim):
    """out is the rounding of the number that it and its low bits make, which
    is therefore within half a bf16 step of it, and no output depends on
    whether the low bits are asked for."""
    pack, q, k, v = problem(q_lengths, k_lengths, heads, kv_heads, dim)
    out, lse, low = kernels.causal_attention_fwd(q, k, v, pack, dim ** -0.5,
                                                 return_low=True)
    again, _ = kernels.causal_attention_fwd(q, k, v, pack, dim ** -0.5)
    assert torch.equal(out, again)
    bits = (out.view(torch.int16).int() << 16) + (low.int() << 8)
    full = bits.view(torch.float32)
    off = (full - out.float()).abs()
    assert (off <= 2.0 ** -8 * out.float().abs()).all()
    seen = out != 0
    assert low[~seen].eq(0).all()
    # Rounding errors are spread evenly over [-128, 128): 255 in 256 are not
    # zero, and the mean of n is within 5 * 74 / sqrt(n) of it. (Rows of one
    # key are exact: a tenth of them and more is left out of account.)
    assert low[seen].ne(0).float().mean() > 0.9
    mean = float(low[seen].float().mean())
    assert abs(mean) < 5 * 74 / int(seen.sum()) ** 0.5 + 0.5


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('q_lengths, k_lengths, heads, kv_heads', [
    ([300, 1, 70], None, 4, 2), ([70, 5], [6000, 3001], 8, 2),
    ([40, 200], [90, 30], 3, 1)])
def test_gradients_of_peaked_weights(q_lengths, k_lengths, heads, kv_heads,
                                     dim):
    """Where a key holds nearly all of a row's weight, dP and D cancel, and the
    rounding of out to bf16 is the largest error of dQ and dK (D's: 2^-8 |out
    dout| against a sum that is a fraction of it). The low bits take it away:
    with them the gradients are nearer to the definition's than without."""
    scale = 4 * dim ** -0.5
    pack, q, k, v = problem(q_lengths, k_lengths, heads, kv_heads, dim)
    dout = rows(pack.total_q, heads, dim, 9)
    grads = gradients(pack, q, k, v, dout, scale)
    check_gradients(pack, q, k, v, dout, grads, scale)
    out, lse, low = kernels.causal_attention_fwd(q, k, v, pack, scale,
                                                 return_low=True)
    exact = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v)]
    for at, keys, h, hk, sees in each_head(pack, q, k):
        qb, kb, vb = q[at, h].double(), k[keys, hk].double(), v[
            keys, hk].double()
        if 0 in (qb.shape[0], kb.shape[0]):
            continue
        g = dout[at, h].double()
        p, _ = softmax64(qb, kb, sees, scale)
        ds = p * (g @ vb.T - (g * (p @ vb)).sum(-1, keepdim=True))
        exact[0][at, h] += scale * ds @ kb
        exact[1][keys, hk] += scale * ds.T @ qb
        exact[2][keys, hk] += p.T @ g
    rounded = kernels.causal_attention_bwd(q, k, v, out, dout, lse, pack,
                                           scale)

    def off(got):
        return [float((a.double() - b).norm() / b.norm())
                for a, b in zip(got, exact)]
    with_low, without = off(grads), off(rounded)
    assert with_low[0] < without[0] and with_low[1] < without[1]
    assert with_low[2] == without[2]


def test_gradients_of_shared_broadcast_and_single_inputs():
    pack, q, _, _ = problem([90, 40], None, 4, 2, 64)
    dout = rows(130, 4, 64, 9)
    k1, v = rows(130, 1, 64, 4), rows(130, 2, 64, 5)
    full = gradients(pack, q, k1.expand(130, 2, 64), v, dout)
    leaf = k1.clone().requires_grad_(True)
    out = kernels.causal_attention(q, leaf.expand(130, 2, 64), v, pack)
    (got,) = torch.autograd.grad(out, leaf, dout)
    assert torch.equal(got, full[1].sum(1, keepdim=True))
    leaf = v.clone().requires_grad_(True)
    out = kernels.causal_attention(q, k1.expand(130, 2, 64), leaf, pack)
    out.backward(dout)
    assert torch.equal(leaf.grad, full[2])
    # Gradients without strides of their own (that of a sum; one row's).
    row = rows(1, 1, 64, 8)
    leaves = [t.clone().requires_grad_(True) for t in (q, v, v)]
    got = torch.autograd.grad(kernels.causal_attention(*leaves, pack), leaves,
                              row.expand(130, 4, 64))
    want = gradients(pack, q, v, v, row.expand(130, 4, 64).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaves = [t.clone().requires_grad_(True) for t in (q, v, v)]
    ones = torch.ones_like(dout)
    got = torch.autograd.grad(kernels.causal_attention(*leaves, pack).sum(),
                              leaves)
    want = gradients(pack, q, v, v, ones)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('heads', [6, 8])
def test_gradients_of_sequences_do_not_reach_one_another(heads, dim):
    pack, q, k, v = problem([150, 70, 33], [150, 200, 33], heads, 2, dim)
    dout = rows(253, heads, dim, 9)
    want = gradients(pack, q, k, v, dout)
    for t in (q, dout):
        t[150:220] = math.nan
    for t in (k, v):
        t[150:350] = math.inf
    got = gradients(pack, q, k, v, dout)
    for a, b, mid in zip(got, want, (220, 350, 350)):
        assert torch.equal(a[:150], b[:150])
        assert torch.equal(a[mid:], b[mid:])


def test_backward_replays_in_a_graph():
    pack, q, k, v = problem([300, 77], None, 4, 2, 128)
    dout = rows(377, 4, 128, 9)
    want = gradients(pack, q, k, v, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            out = kernels.causal_attention(*leaves, pack)
            got = torch.autograd.grad(out, leaves, dout)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_repeats_and_replays():
    pack, q, k, v = problem([500, 120], None, 8, 2, 128)
    want = kernels.causal_attention(q, k, v, pack)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        out = kernels.causal_attention(q, k, v, pack)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    fresh = sequences.SequencePack([500, 120], device=DEV)
    with pytest.raises(RuntimeError, match='before the capture'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            kernels.causal_attention(q, k, v, fresh)


def test_backward_refuses_what_the_forward_did_not_return():
    pack, q, k, v = problem([40, 30], None, 4, 2, 64)
    out, lse, low = kernels.causal_attention_fwd(q, k, v, pack, 0.1,
                                                 return_low=True)
    for o, l, b, match in [(out[:69], lse, low, 'shape of q'),
                           (out, lse[:69], low, 'shape of q'),
                           (out, lse.double(), low, 'fp32'),
                           (out.float(), lse, low, 'bf16'),
                           (out, lse, low[:69], 'low'),
                           (out, lse, low.short(), 'low'),
                           (out, lse, low.transpose(0, 1).contiguous()
                            .transpose(0, 1), 'low'),
                           (out, lse, low.cpu(), 'low')]:
        with pytest.raises(ValueError, match=match):
            kernels.causal_attention_bwd(q, k, v, o, out, l, pack, 0.1, low=b)


@pytest.mark.parametrize('dim', [64, 128])
def test_low_bits_of_values_at_the_ends_of_the_type(dim):
    """One key a row: out is the value row, exactly, whatever its size, and
    NaN and infinity stay what they are."""
    pack, q, k, v = problem([1, 1, 1, 1], None, 2, 1, dim)
    v[0] = torch.finfo(torch.bfloat16).max
    v[1] = -2.0 ** -126
    v[2, 0, :8] = float('inf')
    v[3, 0, 5] = float('nan')
    out, _, low = kernels.causal_attention_fwd(q, k, v, pack, 0.1,
                                               return_low=True)
    for h in range(2):
        assert torch.equal(out[:3, h], v[:3, 0])
        assert out[3, h, 5].isnan() and not out[3, h, 6].isnan()
    full = ((out.view(torch.int16).int() << 16) + (low.int() << 8)).view(
        torch.float32)
    assert torch.equal(full[:3], out[:3].float())
    assert full[3, :, 5].isnan().all()


@pytest.mark.parametrize('dim', [64, 128])
def test_many_short_items_repeat(dim):
    """Items of one block or two: every block loads an item's table entry, so
    the roles of a kernel run at their most uneven."""
    lengths = [1 + (37 * i) % 260 for i in range(900)]
    pack, q, k, v = problem(lengths, None, 8, 4, dim)
    dout = rows(pack.total_q, 8, dim, 9)
    out, lse, low = kernels.causal_attention_fwd(q, k, v, pack, 0.1,
                                                 return_low=True)
    grads = kernels.causal_attention_bwd(q, k, v, out, dout, lse, pack, 0.1,
                                         low=low)
    for _ in range(40):
        again = kernels.causal_attention_fwd(q, k, v, pack, 0.1)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
        again = kernels.causal_attention_bwd(q, k, v, out, dout, lse, pack,
                                             0.1, low=low)
        assert all(torch.equal(a, b) for a, b in zip(again, grads))


def equal_keys(lengths, heads, kv_heads, dim, seed=21):
    """A pack whose sequences repeat one key row, so that a row's weights are
    equal and none is rounded (all are 1 before the division by their sum)."""
    pack, q, k, v = problem(lengths, None, heads, kv_heads, dim, seed)
    first = 0
    for n in lengths:
        k[first:first + n] = k[first:first + 1].clone()
        first += n
    return pack, q, k, v


# At most 64 keys a row: four products of 16 keys, whose 17 terms each may be
# off by 2^-23 of the sum, 4 * 17 * 2^-23 < 2^-16; the weights' 2^-22 and the
# division are inside it.
SHORT = [64, 33, 50, 1, 17]
SHORT_SUM = 2.0 ** -16


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('heads, kv_heads', [(8, 2), (3, 3)])
def test_low_bits_hold_seven_bits_more_than_out(heads, kv_heads, dim):
    """A unit of the low bits is 2^-15 of the number at most, and they are
    half a unit off, a whole one where 128 is held at 127."""
    pack, q, k, v = equal_keys(SHORT, heads, kv_heads, dim)
    v = v.abs()  # no sum cancels
    out, _, low = kernels.causal_attention_fwd(q, k, v, pack, dim ** -0.5,
                                               return_low=True)
    full = ((out.view(torch.int16).int() << 16) + (low.int() << 8)).view(
        torch.float32)
    for at, keys, h, hk, sees in each_head(pack, q, k):
        p = sees.double() / sees.sum(-1, keepdim=True)
        want = p @ v[keys, hk].double()
        err = (full[at, h].double() - want).abs()
        assert (err <= (2.0 ** -15 + SHORT_SUM) * want).all()


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('heads, kv_heads', [(8, 2), (3, 3)])
def test_row_sums_of_the_backward_take_the_low_bits(heads, kv_heads, dim):
    """Value rows that differ by a fiftieth: dP and D nearly cancel, and D may
    be off by what out and its low bits are (2^-15 and the sums' 2^-16, of
    sum |do out|), not by the 2^-8 of out alone. dP and D are sums of D
    products, off by (D + 8) 2^-24 each."""
    scale = dim ** -0.5
    pack, q, k, v = equal_keys(SHORT, heads, kv_heads, dim)
    base = rows(1, kv_heads, dim, 31)
    base = torch.where(base < 0, base - 1, base + 1).float()
    v = (base * (1 + 0.02 * v.float())).bfloat16()
    dout = rows(pack.total_q, heads, dim, 9)
    out, lse, low = kernels.causal_attention_fwd(q, k, v, pack, scale,
                                                 return_low=True)
    want = [torch.zeros(t.shape, dtype=torch.float64, device=DEV)
            for t in (q, k)]
    bound = [torch.zeros_like(t) for t in want]
    u, sums = 2.0 ** -8, 2 * (dim + 8) * 2.0 ** -24
    for at, keys, h, hk, sees in each_head(pack, q, k):
        qb, kb, vb = q[at, h].double(), k[keys, hk].double(), v[
            keys, hk].double()
        g = dout[at, h].double()
        p = sees.double() / sees.sum(-1, keepdim=True)
        o = p @ vb
        size = (qb.abs() @ kb.abs().T).amax(-1, keepdim=True) * scale
        e = 2 * 2.0 ** -24 * (dim + 8) * size + 2.0 ** -14
        ds = p * (g @ vb.T - (g * o).sum(-1, keepdim=True))
        off = (u + e) * ds.abs() + p * (
            (2.0 ** -15 + SHORT_SUM + sums) *
            (g * o).abs().sum(-1, keepdim=True) +
            sums * (g.abs() @ vb.abs().T)) * (1 + u)
        want[0][at, h] += scale * ds @ kb
        want[1][keys, hk] += scale * ds.T @ qb
        bound[0][at, h] += scale * off @ kb.abs()
        bound[1][keys, hk] += scale * off.T @ qb.abs()

    def holds(low):
        got = kernels.causal_attention_bwd(q, k, v, out, dout, lse, pack,
                                           scale, low=low)
        return [bool(((a.double() - w).abs() <= b + u * w.abs() + 1e-30).all())
                for a, w, b in zip(got, want, bound)]
    assert holds(low) == [True, True]
    # The bound tells the two apart.
    assert holds(None)[0] is False


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('heads, kv_heads', [(2, 2), (6, 2), (8, 1)])
@pytest.mark.parametrize('q_lengths, k_lengths', [
    ([1000, 50], None), ([700], [1100])])
def test_how_far_rows_that_are_not_finite_reach(q_lengths, k_lengths, heads,
                                                kv_heads, dim):
    """Rows that do not see a row that is not finite, and are further away
    than 2 (128 // group) + 126 tokens, are what they are without it."""
    reach = 2 * (128 // (heads // kv_heads)) + 126
    pack, q, k, v = problem(q_lengths, k_lengths, heads, kv_heads, dim)
    dout = rows(pack.total_q, heads, dim, 9)
    before = int(pack.k_lengths[0] - pack.q_lengths[0])
    want = kernels.causal_attention(q, k, v, pack)
    want_grads = gradients(pack, q, k, v, dout)
    # A key and its value: the queries before it.
    for key in (before + 384, before + 511, before + 640):
        k_bad, v_bad = k.clone(), v.clone()
        k_bad[key], v_bad[key] = math.inf, math.nan
        out = kernels.causal_attention(q, k_bad, v_bad, pack)
        dq, _, _ = gradients(pack, q, k_bad, v_bad, dout)
        far = key - reach - before  # the first query that it may reach
        assert torch.equal(out[:far], want[:far])
        assert torch.equal(dq[:far], want_grads[0][:far])
        assert out[key - before:q_lengths[0]].isnan().all()
        assert torch.equal(out[q_lengths[0]:], want[q_lengths[0]:])
    # A query and its output's gradient: the keys behind it.
    for query in (0, 127, 256):
        q_bad, dout_bad = q.clone(), dout.clone()
        q_bad[query], dout_bad[query] = math.nan, math.inf
        dq, dk, dv = gradients(pack, q_bad, k, v, dout_bad)
        far = before + query + reach + 1
        for got, ref in ((dk, want_grads[1]), (dv, want_grads[2])):
            assert torch.equal(got[far:], ref[far:])
        other = torch.arange(pack.total_q, device=DEV) != query
        assert torch.equal(dq[other], want_grads[0][other])
