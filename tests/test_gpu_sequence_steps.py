"""The sequence operators together, as a decoder uses them: a prompt, a chunk
behind it and single tokens through `attention.CachedAttention` give what one
causal pass over the whole sequences gives, and a training step goes through
`attention.CausalAttention`.

All three read the same bf16 rows, so two results differ by the roundings of
each: weights 2^-8 of sum_j p_j |v_j| (at most max|v| of the sequence) and
outputs 2^-8, twice.
"""

import pytest
import torch

from miowtion_b200 import _lib
from miowtion_b200 import attention
from miowtion_b200 import kernels
from miowtion_b200 import kvcache
from miowtion_b200 import sequences

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.device_status(reset=True)
    yield
    assert _lib.device_status(reset=True) == 0, 'the status word was set'


def rows(n, heads, dim, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(n, heads, dim, generator=gen).to(DEV, torch.bfloat16)


def steps_of(prompt, chunk, tokens):
    """(first row, rows) of each step of each sequence."""
    out = [([0] * len(prompt), prompt), (prompt, chunk)]
    at = [p + c for p, c in zip(prompt, chunk)]
    for t in range(tokens):
        out.append(([a + t for a in at], [1] * len(at)))
    return out


def caches_and_table(totals, layers, size, kv_heads, dim, storage):
    pages = [-(-n // size) for n in totals]
    table = torch.zeros(len(totals), max(pages), dtype=torch.int32)
    order = torch.randperm(sum(pages), generator=torch.Generator(
    ).manual_seed(1)).to(torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    caches = [kvcache.PagedCache.empty(sum(pages), size, kv_heads, dim,
                                       storage, DEV) for _ in range(layers)]
    return caches, table.to(DEV)


@pytest.mark.parametrize('dim, heads, kv_heads, size', [
    (128, 8, 2, 16), (64, 6, 2, 64)])
def test_prompt_chunk_and_tokens_equal_one_pass(dim, heads, kv_heads, size):
    prompt, chunk, tokens, layers = [130, 5, 64], [40, 1, 100], 3, 2
    totals = [p + c + tokens for p, c in zip(prompt, chunk)]
    caches, table = caches_and_table(totals, layers, size, kv_heads, dim,
                                     'bf16')
    whole = sequences.SequencePack(totals, device=DEV)
    first = whole.q_offsets.tolist()
    for layer in range(layers):
        q = rows(whole.total_q, heads, dim, 10 * layer)
        k, v = (rows(whole.total_q, kv_heads, dim, 10 * layer + i)
                for i in (1, 2))
        want = attention.CausalAttention(whole)(q, k, v, layer)
        got = torch.full_like(want, float('nan'))
        for start, count in steps_of(prompt, chunk, tokens):
            at = torch.cat([torch.arange(f + s, f + s + n) for f, s, n in
                            zip(first, start, count)]).to(DEV)
            pack = sequences.SequencePack(
                count, [s + n for s, n in zip(start, count)], DEV)
            fn = attention.CachedAttention(caches, table, pack)
            got[at] = fn(q[at], k[at], v[at], layer)
        bound = 2 * 2.0 ** -8 * (v.abs().max().float() + want.abs().float())
        assert ((got.float() - want.float()).abs() <= bound).all()


@pytest.mark.parametrize('storage', ['bf16', 'int8', 'e4m3'])
def test_a_captured_decoding_step_advances(storage):
    dim, heads, kv_heads, size, steps = 64, 4, 2, 16, 4
    lengths = [14, 31]
    caches, table = caches_and_table([n + steps for n in lengths], 1, size,
                                     kv_heads, dim, storage)
    twins, _ = caches_and_table([n + steps for n in lengths], 1, size,
                                kv_heads, dim, storage)
    prompt = sequences.SequencePack(lengths, device=DEV)
    k, v = (rows(prompt.total_q, kv_heads, dim, s) for s in (1, 2))
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    for c in (caches[0], twins[0]):
        c.write(k, v, table, zero, prompt)
    news = [[rows(2, h, dim, 30 + 3 * t + i)
             for i, h in enumerate((heads, kv_heads, kv_heads))]
            for t in range(steps)]
    want = []
    for t, qkv in enumerate(news):
        pack = sequences.SequencePack([1, 1], [n + t + 1 for n in lengths],
                                      DEV)
        want.append(attention.CachedAttention(twins, table, pack)(*qkv, 0))
    pack = sequences.SequencePack([1, 1], [n + 1 for n in lengths], DEV)
    fn = attention.CachedAttention(caches, table, pack)
    held = [t.clone() for t in news[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = fn(*held, 0)
        fn.advance()
    torch.cuda.current_stream().wait_stream(side)
    for t, qkv in enumerate(news):
        for dst, src in zip(held, qkv):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[t])


def test_training_step_through_the_attention_function():
    pack = sequences.SequencePack([90, 200, 1], device=DEV)
    fn = attention.CausalAttention(pack, 0.2)
    q = rows(291, 4, 64, 1).requires_grad_(True)
    k, v = (rows(291, 2, 64, s).requires_grad_(True) for s in (2, 3))
    fn(q, k, v, 0).float().square().mean().backward()
    out, lse, low = kernels.causal_attention_fwd(
        q.detach(), k.detach(), v.detach(), pack, 0.2, return_low=True)
    dout = (out.float() * 2 / out.numel()).to(torch.bfloat16)
    want = kernels.causal_attention_bwd(q.detach(), k.detach(), v.detach(),
                                        out, dout, lse, pack, 0.2, low=low)
    assert all(torch.equal(t.grad, w) for t, w in zip((q, k, v), want))


def test_cached_attention_refuses():
    caches, table = caches_and_table([8, 8], 1, 16, 2, 64, 'bf16')
    pack = sequences.SequencePack([2, 3], device=DEV)
    fn = attention.CachedAttention(caches, table, pack)
    with pytest.raises(ValueError, match='single tokens'):
        fn.advance()
    q = rows(5, 4, 64, 1).requires_grad_(True)
    k = rows(5, 2, 64, 1)
    with pytest.raises(ValueError, match='no gradient'):
        fn(q, k, k, 0)
    with pytest.raises(ValueError, match='below'):
        attention.CachedAttention(caches, table, sequences.SequencePack(
            [4, 1], [3, 1], DEV))
