"""The sequence operators, case by case: attention of packed prompts (forward
and training step), the paged key-value cache (rows written, contexts read
back) and attention of single tokens over it.

`run` computes a case with elementary torch operations in fp32, or, where
`own` is true, through the package's entry points: `kernels.causal_attention`,
`kvcache.PagedCache.write`, `.read` and `.attend`.

Definitions, for query row i of a sequence with n queries and c keys (c >= n:
the rows before the queries are its earlier tokens; c < n leaves the first
n - c rows without a key):
    prompt  row i sees keys j <= i + c - n; out_i = sum_j p_ij v_j with
            p = softmax(scale q_i k_j), lse_i = log sum_j exp(scale q_i k_j);
            out 0 and lse -inf without keys
    step    the same with the gradients of sum(out * dout)
    cache   each (token, head) row x of k and v is stored as codes times one
            scale. int8: scale = max|x| / 127, code = round(x * 127 / max|x|).
            e4m3: scale = 2^e, e the smallest integer >= -120 with max|x|
            <= 448 * 2^e, code = x / scale rounded to e4m3. Rounding is to
            nearest, ties to even; an all-zero row has scale 0. bf16: the row
            itself. Read back, a row is code * scale in bf16.
    decode  one query per sequence over its cached rows j < length
"""

import math

import numpy as np
import torch

own = False

DEVICE = 'cuda'
PAGE = 'page_size'
# fp32 elements of one score block of the plain forms (bounds their memory).
_BLOCK = 1 << 28


def listed():
    return [
        # A caption of a few hundred tokens, one head per key head: latency.
        dict(name='prompt_caption', op='prompt', sequences=1, longest=257,
             shortest=257, prefix=0, heads=8, kv_heads=8, dim=128),
        # A batch of ragged captions and prompts, packed, heads in groups of 4.
        dict(name='prompt_ragged', op='prompt', sequences=24, longest=2048,
             shortest=9, prefix=0, heads=32, kv_heads=8, dim=128),
        # A chunk of each request behind an earlier context, narrow heads.
        dict(name='prompt_chunk', op='prompt', sequences=4, longest=1024,
             shortest=500, prefix=7001, heads=14, kv_heads=2, dim=64),
        # A whole clip of 20 x 32 x 56 tokens, causal.
        dict(name='prompt_clip', op='prompt', sequences=1, longest=35840,
             shortest=35840, prefix=0, heads=24, kv_heads=6, dim=128),
        # A training step on a few short samples.
        dict(name='step_short', op='step', sequences=3, longest=300,
             shortest=45, prefix=0, heads=4, kv_heads=2, dim=64),
        # A training step on samples packed to some 14,000 tokens.
        dict(name='step_packed', op='step', sequences=4, longest=8192,
             shortest=1000, prefix=0, heads=16, kv_heads=4, dim=128),
        # Chunks of 16 requests written behind their contexts, which are read
        # back for the attention of the chunk.
        dict(name='cache_chunk', op='cache', storage='e4m3', sequences=16,
             longest=256, shortest=31, prefix=1000, kv_heads=2, dim=64,
             page_size=16),
        # Whole prompts written and read back.
        dict(name='cache_prompt', op='cache', storage='int8', sequences=8,
             longest=16384, shortest=1024, prefix=0, kv_heads=8, dim=128,
             page_size=64),
        # One request's next token.
        dict(name='decode_one', op='decode', storage='e4m3', sequences=1,
             longest=1500, shortest=1500, heads=32, kv_heads=8, dim=128,
             page_size=64),
        # A batch of requests of all lengths.
        dict(name='decode_batch', op='decode', storage='int8', sequences=64,
             longest=8192, shortest=100, heads=32, kv_heads=8, dim=128,
             page_size=16),
        # One key head for all query heads, narrow heads, odd group.
        dict(name='decode_shared', op='decode', storage='bf16', sequences=17,
             longest=4096, shortest=600, heads=7, kv_heads=1, dim=64,
             page_size=32),
        # A few clips' worth of context for each request.
        dict(name='decode_long', op='decode', storage='bf16', sequences=4,
             longest=94624, shortest=35840, heads=48, kv_heads=8, dim=128,
             page_size=128),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['prompt', 'step', 'cache', 'decode'])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 7, 8])
    case = dict(op=op, dim=dim, kv_heads=kv_heads)
    if op in ('prompt', 'step'):
        sequences = _log_int(rng, 1, 24)
        longest = _log_int(rng, 16, 16384 // sequences)
        case.update(heads=heads, sequences=sequences, longest=longest,
                    shortest=_log_int(rng, 1, longest),
                    prefix=rng.choice([0, 0, _log_int(rng, 1, 4096)]))
        if op == 'step':
            case['longest'] = max(1, longest // 2)
            case['shortest'] = min(case['shortest'], case['longest'])
        return case
    case.update(storage=rng.choice(['bf16', 'int8', 'e4m3']),
                page_size=rng.choice([16, 32, 64, 128]))
    if op == 'cache':
        sequences = _log_int(rng, 1, 64)
        longest = _log_int(rng, 1, 32768 // sequences)
        case.update(sequences=sequences, longest=longest,
                    shortest=_log_int(rng, 1, longest),
                    prefix=rng.choice([0, _log_int(rng, 1, 512)]))
        return case
    sequences = _log_int(rng, 1, 128)
    longest = _log_int(rng, 16, 262144 // sequences)
    case.update(heads=heads, sequences=sequences, longest=longest,
                shortest=_log_int(rng, 1, longest))
    return case


def _lengths(case):
    """Lengths spread over the logarithm of [shortest, longest], by the case
    alone; the first is the longest."""
    low, high = case['shortest'], case['longest']
    return [max(1, round(high * (low / high) ** ((i * 0.6180339887) % 1.0)))
            for i in range(case['sequences'])]


def _contexts(case):
    """Keys of each sequence: its own rows and those before them."""
    return [n + (case['prefix'] + 37 * i if case['prefix'] else 0)
            for i, n in enumerate(_lengths(case))]


def _offsets(lengths):
    return [0] + np.cumsum(lengths).tolist()


def _scale(case):
    return case['dim'] ** -0.5


def _rows(gen, n, heads, dim, spread=0.0):
    """N(0, 1) rows; keys have channels of unequal size (`spread`)."""
    x = torch.randn(n, heads, dim, generator=gen, device=DEVICE)
    if spread:
        x *= torch.exp(spread * torch.randn(heads, dim, generator=gen,
                                            device=DEVICE))
    return x.to(torch.bfloat16)


# ---------------------------------------------------------------------------
# codes of the cache, plain form
# ---------------------------------------------------------------------------

_CODE = {'int8': torch.int8, 'e4m3': torch.float8_e4m3fn}


def _power_of_two(e):
    return ((e + 127) << 23).view(torch.float32)


def _encode(x, storage):
    """(codes, scales) of rows x [..., D] (bf16 rows: themselves, None)."""
    if storage == 'bf16':
        return x, None
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    if storage == 'int8':
        # 64 bits: a quotient next to a half must not be rounded onto it.
        codes = torch.round(x.double() * 127.0 / top.double().clamp_min(1e-300))
        scale = top / 127.0
    else:
        mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent
        # top <= 448 * 2^e = 0.875 * 2^(9 + e)
        e = (exponent - 9 + (mantissa > 0.875).int()).clamp_min(-120)
        codes = x * _power_of_two(-e)
        scale = torch.where(top == 0, torch.zeros_like(top), _power_of_two(e))
    return codes.to(_CODE[storage]), scale.squeeze(-1)


def _paged(case, gen, contexts):
    """A cache whose pages lie in any order, with the contexts' rows in it;
    the pages' rows behind a context keep what was there before."""
    page, kv_heads, dim = case[PAGE], case['kv_heads'], case['dim']
    counts = [-(-c // page) for c in contexts]
    total = sum(counts) + 3
    order = torch.randperm(total, generator=gen, device=DEVICE)[:sum(counts)]
    table = torch.zeros(len(contexts), max(counts), dtype=torch.int32,
                        device=DEVICE)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    store = {'table': table}
    for name, spread in (('k', 0.5), ('v', 0.0)):
        rows = _rows(gen, total * page, kv_heads, dim, spread)
        rows = rows.view(total, page, kv_heads, dim).transpose(1, 2)
        codes, scales = _encode(rows, case['storage'])
        store[name] = codes.contiguous()
        store[name + '_scale'] = (None if scales is None
                                  else scales.contiguous())
    return store


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = dict(case=case)
    if case['op'] in ('prompt', 'step'):
        lengths, contexts = _lengths(case), _contexts(case)
        n, c = sum(lengths), sum(contexts)
        state['q'] = _rows(gen, n, case['heads'], case['dim'])
        state['k'] = _rows(gen, c, case['kv_heads'], case['dim'], 0.5)
        state['v'] = _rows(gen, c, case['kv_heads'], case['dim'])
        if case['op'] == 'step':
            state['dout'] = _rows(gen, n, case['heads'], case['dim'])
            if own:
                for name in ('q', 'k', 'v'):
                    state[name].requires_grad_(True)
        if own:
            from miowtion_b200 import sequences
            state['pack'] = sequences.SequencePack(lengths, contexts, DEVICE)
        return state
    contexts = _contexts(case) if case['op'] == 'cache' else _lengths(case)
    state.update(_paged(case, gen, contexts))
    if case['op'] == 'cache':
        lengths = _lengths(case)
        state['new_k'] = _rows(gen, sum(lengths), case['kv_heads'],
                               case['dim'], 0.5)
        state['new_v'] = _rows(gen, sum(lengths), case['kv_heads'],
                               case['dim'])
        state['starts'] = torch.tensor(
            [c - n for c, n in zip(contexts, lengths)], dtype=torch.int32,
            device=DEVICE)
    else:
        state['q'] = _rows(gen, len(contexts), case['heads'], case['dim'])
        state['lengths'] = torch.tensor(contexts, dtype=torch.int32,
                                        device=DEVICE)
    if own:
        from miowtion_b200 import kvcache
        state['cache'] = kvcache.PagedCache(
            state['k'], state['v'], state['k_scale'], state['v_scale'])
        if case['op'] == 'cache':
            from miowtion_b200 import sequences
            state['pack'] = sequences.SequencePack(_lengths(case), contexts,
                                                   DEVICE)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _blocks(case, b, n, c):
    """Row blocks of one sequence: (first row, last row, keys they see)."""
    step = max(1, _BLOCK // max(1, case['heads'] * c))
    for r0 in range(0, n, step):
        r1 = min(n, r0 + step)
        yield r0, r1, max(0, min(c, r1 + c - n))


def _scores(case, q, k, r0, r1, shift):
    """Masked scaled scores [kv_heads, group * rows, keys] of rows r0..r1."""
    kv, dim = case['kv_heads'], case['dim']
    group = case['heads'] // kv
    qb = q.reshape(r1 - r0, kv, group, dim).permute(1, 2, 0, 3)
    s = torch.matmul(qb.reshape(kv, -1, dim), k.transpose(1, 2))
    s *= _scale(case)
    rows = torch.arange(r0, r1, device=q.device).repeat(group)
    hidden = torch.arange(k.shape[1], device=q.device) > (rows + shift)[:, None]
    return s.masked_fill_(hidden, -math.inf)


def _ungroup(case, x, rows):
    """[kv_heads, group * rows, ...] -> [rows, heads, ...]."""
    kv = case['kv_heads']
    x = x.reshape(kv, case['heads'] // kv, rows, *x.shape[2:])
    x = x.movedim(2, 0)
    return x.reshape(rows, case['heads'], *x.shape[3:])


def _softmax(s):
    """Weights that sum to 1 (0 without keys) and the log-sum-exp."""
    if s.shape[2] == 0:
        return s, torch.full(s.shape[:2], -math.inf, device=s.device)
    top = s.amax(-1, keepdim=True)
    safe = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(safe).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (safe + total.log()).squeeze(-1)
    return p.div_(torch.where(total == 0, torch.ones_like(total), total)), lse


def _run_prompt(state, grads):
    case = state['case']
    lengths, contexts = _lengths(case), _contexts(case)
    q0, k0 = _offsets(lengths), _offsets(contexts)
    q, k, v = (state[x].float() for x in ('q', 'k', 'v'))
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, device=q.device)
    if grads:
        dout = state['dout'].float()
        dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    kv, dim = case['kv_heads'], case['dim']
    group = case['heads'] // kv
    for b, (n, c) in enumerate(zip(lengths, contexts)):
        kb = k[k0[b]:k0[b + 1]].transpose(0, 1)
        vb = v[k0[b]:k0[b + 1]].transpose(0, 1)
        for r0, r1, seen in _blocks(case, b, n, c):
            at = slice(q0[b] + r0, q0[b] + r1)
            p, l = _softmax(_scores(case, q[at], kb[:, :seen], r0, r1, c - n))
            o = torch.matmul(p, vb[:, :seen])
            out[at] = _ungroup(case, o, r1 - r0)
            lse[at] = _ungroup(case, l, r1 - r0)
            if not grads:
                continue
            do = dout[at].reshape(r1 - r0, kv, group, dim).permute(1, 2, 0, 3)
            do = do.reshape(kv, -1, dim)
            qb = q[at].reshape(r1 - r0, kv, group, dim).permute(1, 2, 0, 3)
            qb = qb.reshape(kv, -1, dim)
            keys = slice(k0[b], k0[b] + seen)
            dv[keys] += torch.matmul(p.transpose(1, 2), do).transpose(0, 1)
            ds = torch.matmul(do, vb[:, :seen].transpose(1, 2))
            ds = (ds - (do * o).sum(-1, keepdim=True)).mul_(p)
            dk[keys] += torch.matmul(ds.transpose(1, 2),
                                     qb).transpose(0, 1) * _scale(case)
            dq[at] = _ungroup(case, torch.matmul(ds, kb[:, :seen]),
                              r1 - r0) * _scale(case)
    if not grads:
        return out.to(torch.bfloat16), lse
    return tuple(x.to(torch.bfloat16) for x in (out, dq, dk, dv))


def _fetch(state, name, b, length):
    """Rows [kv_heads, length, D] in fp32 of one sequence's context."""
    case = state['case']
    pages = state['table'][b, :-(-length // case[PAGE])].long()
    x = state[name][pages].float()
    if state[name + '_scale'] is not None:
        x = x * state[name + '_scale'][pages][..., None]
    x = x.transpose(0, 1).reshape(case['kv_heads'], -1, case['dim'])
    return x[:, :length]


def _run_cache(state):
    case = state['case']
    lengths, contexts = _lengths(case), _contexts(case)
    offsets = _offsets(lengths)
    for b, (n, c) in enumerate(zip(lengths, contexts)):
        place = torch.arange(c - n, c, device=DEVICE)
        page = state['table'][b].long()[place // case[PAGE]]
        slot = place % case[PAGE]
        for name in ('k', 'v'):
            rows = state['new_' + name][offsets[b]:offsets[b + 1]]
            codes, scales = _encode(rows, case['storage'])
            target = state[name]
            if target.dtype == torch.float8_e4m3fn:
                target, codes = target.view(torch.uint8), codes.view(torch.uint8)
            target[page, :, slot] = codes
            if scales is not None:
                state[name + '_scale'][page, :, slot] = scales
    return tuple(torch.cat([_fetch(state, name, b, c).transpose(0, 1)
                            for b, c in enumerate(contexts)])
                 .to(torch.bfloat16) for name in ('k', 'v'))


def _run_decode(state):
    case = state['case']
    kv, dim = case['kv_heads'], case['dim']
    outs, lses = [], []
    for b, length in enumerate(_lengths(case)):
        q = state['q'][b].float().reshape(kv, -1, dim)
        s = torch.matmul(q, _fetch(state, 'k', b, length).transpose(1, 2))
        p, lse = _softmax(s.mul_(_scale(case)))
        outs.append(torch.matmul(p, _fetch(state, 'v', b, length))
                    .reshape(-1, dim))
        lses.append(lse.reshape(-1))
    return torch.stack(outs).to(torch.bfloat16), torch.stack(lses)


def _run_own(state):
    op = state['case']['op']
    if op in ('prompt', 'step'):
        from miowtion_b200 import kernels
        if op == 'prompt':
            return kernels.causal_attention(state['q'], state['k'],
                                            state['v'], state['pack'],
                                            return_lse=True)
        leaves = state['q'], state['k'], state['v']
        out = kernels.causal_attention(*leaves, state['pack'])
        return (out.detach(),
                *torch.autograd.grad(out, leaves, state['dout']))
    cache = state['cache']
    if op == 'cache':
        cache.write(state['new_k'], state['new_v'], state['table'],
                    state['starts'], state['pack'])
        return cache.read(state['table'], state['pack'])
    return cache.attend(state['q'], state['table'], state['lengths'],
                        return_lse=True)


def run(state):
    if own:
        return _run_own(state)
    op = state['case']['op']
    if op in ('prompt', 'step'):
        return _run_prompt(state, op == 'step')
    return _run_cache(state) if op == 'cache' else _run_decode(state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------


def work(case):
    dim, kv = case['dim'], case['kv_heads']
    if case['op'] in ('prompt', 'step'):
        lengths, contexts = _lengths(case), _contexts(case)
        # Rows 0 .. n - 1 see c - n + 1 .. c keys (here always c >= n).
        pairs = sum(n * (c - n) + n * (n + 1) // 2
                    for n, c in zip(lengths, contexts)) * case['heads']
        q = sum(lengths) * case['heads']
        k = sum(contexts) * kv
        if case['op'] == 'prompt':
            return {'bytes': 2 * dim * (2 * q + 2 * k) + 4 * q,
                    'flops': 4 * dim * pairs}
        return {'bytes': 2 * dim * (4 * q + 4 * k), 'flops': 14 * dim * pairs}
    width = dim * 2 if case['storage'] == 'bf16' else dim + 4
    if case['op'] == 'cache':
        new = sum(_lengths(case)) * kv * 2
        all_rows = sum(_contexts(case)) * kv * 2
        # New rows come from the call, so only the others are read back; every
        # row of the contexts goes out in bf16.
        return {'bytes': new * (2 * dim + width) +
                (all_rows - new) * width + all_rows * 2 * dim,
                'flops': (3 * new + all_rows) * dim}
    rows = sum(_lengths(case))
    q = case['sequences'] * case['heads']
    return {'bytes': rows * kv * 2 * width + q * (4 * dim + 4),
            'flops': 4 * dim * rows * case['heads']}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _grid64(x, storage):
    """Rows x [..., D] (fp64) as the cache holds them, in real arithmetic."""
    top = x.abs().amax(-1, keepdim=True)
    if storage == 'bf16':
        return x
    if storage == 'int8':
        # The scale is held in fp32.
        held = (top / 127).float().double()
        return torch.where(top > 0, (x * 127 / top).round() * held, 0 * x)
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448)).clamp_min(-120)
    e = torch.where(top <= 448 * 2.0 ** (e - 1), (e - 1).clamp_min(-120), e)
    e = torch.where(top > 448 * 2.0 ** e, e + 1, e)
    y = x / 2.0 ** e
    # Steps of e4m3: 2^-3 of the value's power of two, 2^-9 below 2^-6.
    power = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
    step = 2.0 ** (power - 3)
    return (y / step).round() * step * 2.0 ** e


def _exact_attend(q, k, v, shift, scale):
    """fp64 attention of q [n, D] over k, v [c, D]; row i sees keys
    <= i + shift. Returns out, lse, weights."""
    s = scale * (q @ k.T)
    sees = (torch.arange(k.shape[0], device=q.device)[None, :] -
            torch.arange(q.shape[0], device=q.device)[:, None]) <= shift
    s = torch.where(sees, s, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(sees, torch.exp(s - lse[:, None]), 0.0)
    return p @ v, lse, p


def exact(case, seed):
    op, dim, kv = case['op'], case['dim'], case['kv_heads']
    state = prepare(case, seed)
    scale = 1.0 / math.sqrt(dim)
    if op in ('prompt', 'step'):
        lengths, contexts = _lengths(case), _contexts(case)
        group = case['heads'] // kv
        q, k, v = (state[x].detach().double() for x in ('q', 'k', 'v'))
        out = torch.zeros_like(q)
        lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
        dout = state['dout'].double() if op == 'step' else None
        dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
        i0 = j0 = 0
        for n, c in zip(lengths, contexts):
            for h in range(case['heads']):
                kb, vb = k[j0:j0 + c, h // group], v[j0:j0 + c, h // group]
                for r in range(0, n, 8192):
                    rows = slice(i0 + r, i0 + min(n, r + 8192))
                    o, l, p = _exact_attend(q[rows, h], kb, vb, c - n + r,
                                            scale)
                    out[rows, h], lse[rows, h] = o, l
                    if op == 'prompt':
                        continue
                    g = dout[rows, h]
                    ds = p * (g @ vb.T - (g * o).sum(-1, keepdim=True))
                    dq[rows, h] = scale * (ds @ kb)
                    dk[j0:j0 + c, h // group] += scale * (ds.T @ q[rows, h])
                    dv[j0:j0 + c, h // group] += p.T @ g
            i0, j0 = i0 + n, j0 + c
        return (out, lse) if op == 'prompt' else (out, dq, dk, dv)
    page, table = case[PAGE], state['table'].cpu()

    def context(name, b, length):
        rows = []
        for at in range(0, length, page):
            number = int(table[b, at // page])
            x = state[name][number].double()
            if state[name + '_scale'] is not None:
                x = x * state[name + '_scale'][number].double()[..., None]
            rows.append(x[:, :length - at])
        return torch.cat(rows, 1)

    if op == 'cache':
        outs = []
        for name in ('k', 'v'):
            parts, at = [], 0
            for b, (n, c) in enumerate(zip(_lengths(case), _contexts(case))):
                x = context(name, b, c).transpose(0, 1).clone()
                new = state['new_' + name][at:at + n].double()
                x[c - n:] = _grid64(new, case['storage'])
                parts.append(x)
                at += n
            outs.append(torch.cat(parts))
        return tuple(outs)
    out = torch.zeros(case['sequences'], case['heads'], dim,
                      dtype=torch.float64, device=DEVICE)
    lse = torch.zeros(out.shape[:2], dtype=torch.float64, device=DEVICE)
    group = case['heads'] // kv
    for b, length in enumerate(_lengths(case)):
        k, v = context('k', b, length), context('v', b, length)
        for h in range(kv):
            heads = slice(h * group, (h + 1) * group)
            o, l, _ = _exact_attend(state['q'][b, heads].double(), k[h], v[h],
                                    length, scale)
            out[b, heads], lse[b, heads] = o, l
    return out, lse
