"""The cases that the per-request operators of a decode step are timed and checked on.

Two operators, both reached through the device ABI (include/glmvx.h):

  lora    glmvx_lora_add: y[t] += scale_a * B_a (A_a x[t]) for the adapter a = ids[t] of each
          token (-1: none, the row stays), added to a shared projection's output y
  select  glmvx_logits_select: per row of logits, repetition / presence / frequency penalties
          from the row's token history, per-token biases, a grammar mask, and the largest
          remaining token

`run` computes a case in elementary torch operations where `own` is false and with the
library's kernels where it is true.  Widths are those of the GLM-MoE-DSA configuration that
bench.py decodes (hidden 6144, q_lora 2048, 64 heads x 256, latent 512 + 64, dense MLP 12288,
vocabulary 154880) and odd ones.
"""
import functools
import math
import os
import sys

import torch

own = False

KINDS = {'f32': (0, torch.float32, 4), 'f16': (1, torch.float16, 2), 'bf16': (30, torch.bfloat16, 2)}


# ------------------------------------------------------------------ the cases
def _lora(name, tokens, rows, cols, adapters, used, max_rank, kind, spread='mixed', none=0, pad=0, even=True):
    """`used` of the bank's `adapters` occur among the tokens; `none` tokens have no adapter; spread
    'mixed' shuffles the tokens, 'runs' keeps each adapter's tokens together, in uneven lengths;
    `even` false gives the adapters ranks from max_rank down; `pad` columns stand between the rows."""
    return {'name': name, 'op': 'lora', 'tokens': tokens, 'rows': rows, 'cols': cols, 'adapters': adapters,
            'used': used, 'max_rank': max_rank, 'kind': kind, 'spread': spread, 'none': none, 'pad': pad, 'even': even}


def _select(name, rows, vocab, history, bias, masks, pad=0):
    """Rows have histories of up to `history` tokens (the first row's is empty), every second one
    `bias` biased tokens; `masks` is 'none', 'loose' (most tokens stay), 'tight' (about a hundred
    stay) or 'mixed' (rows with and without, one table that leaves nothing)."""
    return {'name': name, 'op': 'select', 'rows': rows, 'vocab': vocab, 'history': history, 'bias': bias,
            'masks': masks, 'pad': pad}


def listed():
    return [
        # one sequence with its adapter on the key/value down-projection: the smallest call, all latency
        _lora('lora 1 token kv_a r8', 1, 576, 6144, 4, 1, 8, 'bf16'),
        # a full decode batch, every request with an adapter of its own, on the query up-projection
        _lora('lora 64 tokens q_b r16', 64, 16384, 2048, 64, 64, 16, 'bf16'),
        # a decode batch that shares a few adapters of unequal ranks, some requests without one
        _lora('lora 48 tokens o_proj r64', 48, 6144, 16384, 12, 5, 64, 'f16', none=9, even=False),
        # odd widths and ranks, f32 adapters, rows inside wider buffers
        _lora('lora 37 tokens odd f32', 37, 1001, 515, 9, 7, 13, 'f32', none=3, pad=5, even=False),
        # prompts of many requests run through the dense MLP's gate together
        _lora('lora 4096 tokens gate r32', 4096, 12288, 6144, 16, 16, 32, 'bf16', spread='runs'),
        # ragged prompts shuffled into one batch, high ranks, some without an adapter
        _lora('lora 1000 tokens q_a r64', 1000, 2048, 6144, 24, 11, 64, 'f16', none=100, even=False),
        # one request alone, a short history, no grammar
        _select('select 1 row', 1, 154880, 300, 8, 'none'),
        # a full decode batch: long histories, biases, grammars on most rows, one of them exhausted
        _select('select 64 rows mixed', 64, 154880, 2048, 300, 'mixed'),
        # a small odd vocabulary inside wider rows
        _select('select 17 rows odd', 17, 32003, 777, 31, 'mixed', pad=13),
        # grammars that leave about a hundred tokens a row
        _select('select 32 rows tight', 32, 154880, 512, 0, 'tight'),
        # the largest: several decode batches' rows at once, loose grammars
        _select('select 256 rows loose', 256, 154880, 1024, 64, 'loose'),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.55:
        tokens = _spread(rng, 1, 4096) if rng.random() < 0.5 else rng.randint(1, 64)
        rows, cols = _spread(rng, 64, 16384), _spread(rng, 64, 16384)
        if rng.random() < 0.6:  # widths of projections are mostly multiples of 64
            rows, cols = max(64, rows // 64 * 64), max(64, cols // 64 * 64)
        tokens = max(1, min(tokens, 4096 * (2 * 12288 + 6144) // (2 * rows + cols)))
        adapters = _spread(rng, 1, 64)
        none = rng.choice([0, 0, tokens // 7])
        used = max(1, min(adapters, rng.randint(1, adapters), tokens - none))
        case = _lora('', tokens, rows, cols, adapters, used, _spread(rng, 1, 64), rng.choice(list(KINDS)),
                     rng.choice(['mixed', 'runs']), none, rng.choice([0, 0, 4, 7]), rng.random() < 0.5)
    else:
        vocab = _spread(rng, 500, 160000)
        rows = min(_spread(rng, 1, 256), 256 * 154880 // vocab)
        case = _select('', rows, vocab, _spread(rng, 1, 4096), rng.choice([0, 5, 64, 300]),
                       rng.choice(['none', 'loose', 'tight', 'mixed']), rng.choice([0, 0, 3, 16]))
    del case['name']
    return case


# ------------------------------------------------------------------ what a case holds
def _ranks(case):
    r, n = case['max_rank'], case['adapters']
    return [r if case['even'] else max(1, r - (i * r) // (n + 1)) for i in range(n)]


def _counts(case):
    """Tokens of each of the used adapters."""
    t, used = case['tokens'] - case['none'], case['used']
    if case['spread'] == 'mixed':
        return [t // used + (i < t % used) for i in range(used)]
    at = [max(i, int(t * (i / used) ** 1.5)) for i in range(used)] + [t]  # uneven runs, one token at least
    return [b - a for a, b in zip(at, at[1:])]


def _lens(case):
    return [case['history'] * i // max(1, case['rows'] - 1) if case['rows'] > 1 else case['history']
            for i in range(case['rows'])]


def _mask_rows(case):
    """The mask table's row of each row of logits (-1: none)."""
    if case['masks'] == 'none':
        return [-1] * case['rows']
    if case['masks'] == 'mixed':
        return [b % 5 - 1 for b in range(case['rows'])]
    return [b % 4 for b in range(case['rows'])]


def work(case):
    if case['op'] == 'lora':
        counts, ranks, size = _counts(case), _ranks(case), KINDS[case['kind']][2]
        tokens, wide = sum(counts), case['rows'] + case['cols']
        return {'bytes': 4 * tokens * (case['cols'] + 2 * case['rows']) + 4 * case['tokens'] +
                sum(r * wide * size for r, c in zip(ranks, counts) if c),
                'flops': sum(2 * c * r * wide for r, c in zip(ranks, counts))}
    rows, vocab = case['rows'], case['vocab']
    words = len(set(m for m in _mask_rows(case) if m >= 0)) * ((vocab + 31) // 32)
    return {'bytes': 8 * rows * vocab + 4 * words + 4 * sum(_lens(case)) + 8 * case['bias'] * ((rows + 1) // 2) +
            40 * rows, 'flops': 6 * rows * vocab}


def prepare(case, seed):
    g = torch.Generator('cuda').manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device='cuda')

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device='cuda')

    s = dict(case)
    if case['op'] == 'lora':
        t, rows, cols, n, r, pad = (case[k] for k in ('tokens', 'rows', 'cols', 'adapters', 'max_rank', 'pad'))
        kind, dtype, _ = KINDS[case['kind']]
        names = torch.randperm(n, generator=g, device='cuda')[:case['used']]
        ids = torch.repeat_interleave(names, torch.tensor(_counts(case), device='cuda'))
        ids = torch.cat([ids, torch.full((case['none'],), -1, device='cuda')])
        if case['spread'] == 'mixed':
            ids = ids[torch.randperm(t, generator=g, device='cuda')]
        ranks = torch.zeros(n, dtype=torch.int32, device='cuda')  # the used adapters take the first ranks
        ranks[names] = whole(_ranks(case)[:case['used']])
        rest = ranks == 0
        ranks[rest] = whole(_ranks(case)[case['used']:])
        s.update(x=normal(t, cols + pad)[:, :cols], y=normal(t, rows + pad)[:, :rows],
                 a=(normal(n, r, cols) / math.sqrt(cols)).to(dtype), b=(normal(n, rows, r) / math.sqrt(r)).to(dtype),
                 ids=ids.to(torch.int32), ranks=ranks, scales=0.5 + torch.rand(n, generator=g, device='cuda'),
                 code=kind)
        return s
    rows, vocab, cap = case['rows'], case['vocab'], case['history'] + 4
    lens = _lens(case)
    # token frequencies fall off steeply, so histories repeat tokens
    u = torch.rand(rows, cap, generator=g, device='cuda', dtype=torch.float64)
    s.update(logits=3 * normal(rows, vocab + case['pad'])[:, :vocab], out=torch.empty(rows, vocab, device='cuda'),
             history=(u ** 4 * vocab).to(torch.int32).clamp(max=vocab - 1),
             fed=torch.randint(vocab, (rows,), generator=g, device='cuda', dtype=torch.int32),
             lens=whole(lens), prompts=whole([n // 2 for n in lens]),
             penalties=torch.stack([1 + torch.rand(rows, generator=g, device='cuda'),
                                    torch.rand(rows, generator=g, device='cuda') - 0.25,
                                    torch.rand(rows, generator=g, device='cuda') - 0.25], 1).contiguous(),
             selected=torch.empty(rows, dtype=torch.int32, device='cuda'),
             bias_ids=None, bias_values=None, bias_lens=None, masks=None, mask_rows=None)
    if case['bias']:
        s.update(bias_ids=torch.randint(vocab, (rows, case['bias']), generator=g, device='cuda', dtype=torch.int32),
                 bias_values=20 * normal(rows, case['bias']),
                 bias_lens=whole([case['bias'] * (1 - b % 2) for b in range(rows)]))
    if case['masks'] != 'none':
        words = (vocab + 31) // 32
        few, most = min(0.5, 100 / vocab), 0.9
        share = {'loose': [most] * 4, 'tight': [few] * 4, 'mixed': [most, few, 0.5, 0.0]}[case['masks']]
        keep = torch.rand(4, words, 32, generator=g, device='cuda') < torch.tensor(share, device='cuda')[:, None, None]
        bits = (keep.long() << torch.arange(32, device='cuda')).sum(-1)
        s.update(masks=torch.where(bits >= 2**31, bits - 2**32, bits).to(torch.int32), mask_rows=whole(_mask_rows(case)))
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    if state['op'] == 'lora':
        return _lora_own(state) if own else _lora_plain(state)
    return _select_own(state) if own else _select_plain(state)


def _lora_plain(s):
    """Every adapter's A on every token, all but a token's own set to nothing, then every B."""
    n, r = s['adapters'], s['max_rank']
    h = s['x'] @ s['a'].float().reshape(n * r, s['cols']).T
    at = torch.arange(n, device='cuda')
    keep = (s['ids'][:, None] == at)[:, :, None] & (torch.arange(r, device='cuda') < s['ranks'][:, None])[None]
    h = torch.where(keep, h.reshape(-1, n, r), 0.0) * s['scales'][None, :, None]
    s['y'] += h.reshape(-1, n * r) @ s['b'].float().transpose(1, 2).reshape(n * r, s['rows'])
    return {'y': s['y']}


def _select_plain(s):
    l, vocab = s['logits'], s['vocab']
    rows, cap = s['history'].shape
    dev = l.device
    # the fed token joins the history, where there is room for it
    room = s['lens'] < cap
    at = s['lens'].long().clamp(max=cap - 1)[:, None]
    s['history'].scatter_(1, at, torch.where(room[:, None], s['fed'][:, None], s['history'].gather(1, at)))
    there = torch.arange(cap, device=dev) < (s['lens'] + room)[:, None]
    out = there & (torch.arange(cap, device=dev) >= s['prompts'][:, None])
    ids = s['history'].long()
    seen = torch.zeros(rows, vocab, device=dev).scatter_add_(1, ids, there.float())
    count = torch.zeros(rows, vocab, device=dev).scatter_add_(1, ids, out.float())
    # a fed token without room still counts
    extra = (~room).float()[:, None]
    seen.scatter_add_(1, s['fed'].long()[:, None], extra)
    count.scatter_add_(1, s['fed'].long()[:, None], extra)
    s['lens'] += room
    rep, pres, freq = (p[:, None] for p in s['penalties'].unbind(1))
    l = torch.where(seen > 0, torch.where(l > 0, l / rep, l * rep), l)
    l = l - count * freq
    l = l - (count > 0) * pres
    if s['bias_ids'] is not None:  # of a token's entries the last holds
        k = torch.arange(1, s['bias_ids'].shape[1] + 1, device=dev).expand(rows, -1)
        k = torch.where(k <= s['bias_lens'][:, None], k, 0)
        last = torch.zeros(rows, vocab, dtype=torch.long, device=dev)
        last = last.scatter_reduce(1, s['bias_ids'].long(), k, 'amax')
        l = l + torch.where(last > 0, s['bias_values'].gather(1, (last - 1).clamp(min=0)), 0.0)
    if s['masks'] is not None:
        bits = s['masks'][s['mask_rows'].long().clamp(min=0)]
        allowed = ((bits[:, :, None] >> torch.arange(32, device=dev)) & 1).reshape(rows, -1)[:, :vocab] > 0
        l = torch.where(allowed | (s['mask_rows'] < 0)[:, None], l, -math.inf)
    top = l.amax(1, keepdim=True)
    first = torch.where(l == top, torch.arange(vocab, device=dev), vocab).amin(1)
    s['selected'] = torch.where(top[:, 0] > -math.inf, first, -1).to(torch.int32)
    return {'logits': l, 'selected': s['selected'], 'history': s['history'], 'lens': s['lens']}


@functools.lru_cache(maxsize=None)
def _runtime():
    sys.path.insert(0, os.path.join(os.getcwd(), 'glm-vx_b200'))
    from gpu import runtime
    return runtime


def _at(t):
    return None if t is None else t.data_ptr()


def _lora_own(s):
    rt = _runtime()
    if 'workspace' not in s:  # kept from then on, as a serving loop keeps it
        need = rt.library().glmvx_lora_workspace_bytes(s['tokens'], s['adapters'], s['max_rank'])
        s['workspace'] = torch.empty(need, dtype=torch.uint8, device='cuda')
    x, y, ws = s['x'], s['y'], s['workspace']
    rt.call('glmvx_lora_add', y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), s['ids'].data_ptr(), s['code'],
            s['a'].data_ptr(), s['b'].data_ptr(), s['ranks'].data_ptr(), s['scales'].data_ptr(), s['tokens'], s['rows'],
            s['cols'], s['adapters'], s['max_rank'], ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    return {'y': y}


def _select_own(s):
    rt = _runtime()
    rt.call('glmvx_logits_select', s['selected'].data_ptr(), s['out'].data_ptr(), s['out'].stride(0),
            s['logits'].data_ptr(), s['logits'].stride(0), s['rows'], s['vocab'], s['fed'].data_ptr(),
            s['history'].data_ptr(), s['history'].shape[1], s['lens'].data_ptr(), s['prompts'].data_ptr(),
            s['penalties'].data_ptr(), _at(s['bias_ids']), _at(s['bias_values']), _at(s['bias_lens']), s['bias'],
            _at(s['masks']), _at(s['mask_rows']), 0 if s['masks'] is None else s['masks'].shape[0],
            torch.cuda.current_stream().cuda_stream)
    return {'logits': s['out'], 'selected': s['selected'], 'history': s['history'], 'lens': s['lens']}


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'lora':
        y, x = s['y'].double(), s['x'].double()
        for i, (r, scale) in enumerate(zip(s['ranks'].tolist(), s['scales'].tolist())):
            mine = (s['ids'] == i).nonzero()[:, 0]
            if len(mine):
                low = torch.einsum('tc,rc->tr', x[mine], s['a'][i, :r].double())
                y[mine] += scale * torch.einsum('tr,nr->tn', low, s['b'][i, :, :r].double())
        return {'y': y}
    got = torch.empty(case['rows'], case['vocab'], dtype=torch.float64, device='cuda')
    lens, prompts, fed = s['lens'].tolist(), s['prompts'].tolist(), s['fed'].tolist()
    mask_rows = s['mask_rows'].tolist() if s['masks'] is not None else [-1] * case['rows']
    for b in range(case['rows']):
        l = s['logits'][b].double()
        rep, pres, freq = s['penalties'][b].double()
        told = s['history'][b, :lens[b]].tolist() + [fed[b]]
        seen = torch.tensor(sorted(set(told)), device='cuda')
        l[seen] = torch.where(l[seen] > 0, l[seen] / rep, l[seen] * rep)
        new, count = torch.tensor(told[prompts[b]:], device='cuda').unique(return_counts=True)
        l[new] -= count * freq + pres
        if s['bias_ids'] is not None:
            n = int(s['bias_lens'][b])
            by = dict(zip(s['bias_ids'][b, :n].tolist(), s['bias_values'][b, :n].tolist()))
            if by:
                l[list(by)] += torch.tensor(list(by.values()), dtype=torch.float64, device='cuda')
        if mask_rows[b] >= 0:
            words = s['masks'][mask_rows[b]].long()
            v = torch.arange(case['vocab'], device='cuda')
            l[(words[v // 32] >> (v % 32)) & 1 == 0] = -math.inf
        got[b] = l
    # the chosen token is a matter of the rounded logits; the state is of whole numbers
    return {'logits': got, 'selected': None, 'history': None, 'lens': None}
