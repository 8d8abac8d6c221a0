"""The operators of a transformer layer that is served in 8-bit integers, as measurable cases.

A case is a dict of plain values; `op` names the operator:

  norm       n2d2b_rmsnorm_quantize: residual sum, root-mean-square norm, 8-bit codes with a scale for each token
  matmul     n2d2b_matmul_i8: 8-bit codes x 8-bit weights with scales for each token and each output channel
  append     n2d2b_kv_append: new keys and values into a paged cache of 8-bit codes with a scale for each page and head
  attention  n2d2b_kv_attention: attention of new tokens over that cache

With `own` false the operators run in their plain form: elementary torch operations in 32 bits.  Codes are returned as
the values they stand for (code x scale); the conversion, one torch operation, is part of the pass on both sides.

Lengths of a batch are a matter of the case and not of the seed, which draws the values.
"""
import math
import random

import torch

own = False

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
TINY = 2.0 ** -100      # a largest magnitude up to this counts as zero: its reciprocal is not held in 32 bits


def _norm(rows, columns, dtype='bf16', residual=True):
    return dict(op='norm', rows=rows, columns=columns, dtype=dtype, residual=residual)


def _matmul(m, n, k, dtype='bf16', bias=False):
    return dict(op='matmul', m=m, n=n, k=k, dtype=dtype, bias=bias)


def _append(batch, new, context, kv_heads=8, head_size=128, page=64, dtype='bf16'):
    return dict(op='append', batch=batch, new=new, context=context, heads=kv_heads, kv_heads=kv_heads, head_size=head_size, page=page,
                dtype=dtype)


def _attention(batch, new, context, heads=32, kv_heads=8, head_size=128, page=64, dtype='bf16', window=0, causal=True):
    return dict(op='attention', batch=batch, new=new, context=context, heads=heads, kv_heads=kv_heads, head_size=head_size, page=page,
                dtype=dtype, window=window, causal=causal)


def listed():
    return [dict(c, name=name) for name, c in (
        # the norm ahead of a projection while eight conversations are answered a token at a time: latency
        ('norm_decode_8x4096', _norm(8, 4096)),
        # the same over the tokens of a batch of prompts: bandwidth
        ('norm_prompt_8192x4096', _norm(8192, 4096)),
        # one token through a square projection: the weights are read once for a single row
        ('matmul_1x4096x4096', _matmul(1, 4096, 4096)),
        # a serving step of 48 conversations through the joint projection to queries, keys and values (32 + 8 + 8 heads of 128)
        ('matmul_48x6144x4096', _matmul(48, 6144, 4096)),
        # a ResNet-50 classifier (2048 features, 1000 classes) over a batch of 1024 with a bias and 32-bit scores: odd width
        ('matmul_classifier_1024x1000x2048', _matmul(1024, 1000, 2048, dtype='f32', bias=True)),
        # prompts through a square projection: the tensor pipe
        ('matmul_4096x4096x4096', _matmul(4096, 4096, 4096, dtype='f16')),
        # 64 conversations each gain a token: every page touched has its scale looked at and, if it grows, its codes rescaled
        ('append_decode_64', _append(64, 1, 200)),
        # prompts of up to 4000 tokens enter the cache, ragged lengths that end inside a page
        ('append_prompt_4x4000', _append(4, 4000, 4000)),
        # one conversation of a small model just begun: latency
        ('attention_decode_1x100', _attention(1, 1, 100, heads=8, kv_heads=2, head_size=64, page=16, dtype='f16')),
        # one long conversation: the cached tokens of eight heads have to be spread over the whole GPU
        ('attention_decode_1x65000', _attention(1, 1, 65000)),
        # a serving step of 48 conversations of up to 8000 tokens
        ('attention_decode_48x8000', _attention(48, 1, 8000)),
        # a piece of a prompt over what the cache holds of it, itself included
        ('attention_prompt_4096_of_8192', _attention(1, 4096, 8192)),
    )]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'matmul', 'matmul', 'append', 'attention', 'attention', 'attention'])
    if op == 'norm':
        columns = rng.choice([512, 1000, 1024, 2048, 4096, 5120, 8192, rng.randrange(64, 8200)])
        return _norm(_log_int(rng, 1, 8192 * 4096 // columns), columns, rng.choice(['bf16', 'bf16', 'f16', 'f32']), rng.random() < 0.7)
    if op == 'matmul':
        n = rng.choice([1000, 1024, 4096, 6144, _log_int(rng, 64, 8192)])
        k = rng.choice([512, 2048, 4096, 16 * _log_int(rng, 4, 512), _log_int(rng, 64, 8192)])
        m = _log_int(rng, 1, min(8192, 4096 ** 3 // (n * k)))
        return _matmul(m, n, k, rng.choice(['bf16', 'bf16', 'f16', 'f32']), rng.random() < 0.3)
    kv_heads, head_size = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    page, dtype = rng.choice([16, 32, 64, 64, 128]), rng.choice(['bf16', 'bf16', 'f16'])
    if op == 'append':
        new = rng.choice([1, 1, _log_int(rng, 2, 4000)])
        batch = _log_int(rng, 1, min(256, 16000 // new))
        return _append(batch, new, min(4000, new + _log_int(rng, 1, 400)), kv_heads, head_size, page, dtype)
    heads = kv_heads * rng.choice([1, 2, 4, 4, 8])
    window, causal = (_log_int(rng, 16, 4096) if rng.random() < 0.2 else 0), True
    if rng.random() < 0.5:
        context = _log_int(rng, 16, 65000)
        batch = _log_int(rng, 1, max(1, min(128, 390000 // context)))
        new = rng.choice([1, 1, 1, rng.randrange(2, 9)])
    else:
        new = _log_int(rng, 9, 4096)
        context = new + rng.choice([0, rng.randrange(0, 4097)])
        batch = max(1, min(8, 20_000_000 // (new * context)))
        if rng.random() < 0.15:
            causal, window = False, 0
    most = 32 * 4096 * 8192 // heads
    if batch * new * context > most:
        batch, new = 1, min(new, most // context)
    return _attention(batch, new, context, heads, kv_heads, head_size, page, dtype, window, causal)


def _lengths(case):
    """(total lengths, new tokens) of the sequences of a batch; the first one has the most, one in sixteen is an idle place."""
    rng = random.Random('%(batch)d %(new)d %(context)d' % case)
    lengths, news = [case['context']], [case['new']]
    for b in range(1, case['batch']):
        if rng.random() < 1 / 16:
            lengths.append(0)
            news.append(0 if case['new'] > 1 else 1)
            continue
        new = 1 if case['new'] == 1 else rng.randrange(1, case['new'] + 1)
        news.append(new)
        lengths.append(rng.randrange(max(new, case['context'] // 4), case['context'] + 1))
    return lengths, news


def _geometry(case):
    """Pages of each sequence, all pages of the pool, entries of a row of the page table."""
    lengths, _ = _lengths(case)
    pages = [max(1, -(-n // case['page'])) for n in lengths]
    return pages, sum(pages) + 3, -(-case['context'] // case['page'])


def _pool(case, pages, gen):
    """A cache in use: values of a normal distribution whose width differs from head to head, 8 bits with a scale for each page and head."""
    shape = (pages, case['kv_heads'], case['page'], case['head_size'])
    width = torch.rand((1, shape[1], 1, 1), device='cuda', generator=gen) + 0.5
    codes = torch.empty(shape, dtype=torch.int8, device='cuda')
    scales = torch.empty(shape[:2], device='cuda')
    for at in range(0, pages, 256):
        x = torch.randn((min(256, pages - at),) + shape[1:], device='cuda', generator=gen) * width
        largest = x.abs().amax((2, 3))
        scales[at:at + 256] = largest / 127
        codes[at:at + 256] = (x * (127 / largest)[:, :, None, None]).round().to(torch.int8)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    state = {'case': case, 'stream': torch.cuda.current_stream().cuda_stream}
    dtype = TYPES[case['dtype']]

    def normal(*shape):
        return torch.randn(shape, device='cuda', generator=gen)

    if case['op'] == 'norm':
        rows, columns = case['rows'], case['columns']
        # a few channels are much larger than the others, as in the residual stream of a trained model
        wide = torch.where(torch.rand(columns, device='cuda', generator=gen) < 0.005, 20.0, 1.0)
        state['x'] = (normal(rows, columns) * wide).to(dtype)
        if case['residual']:
            state['residual'] = normal(rows, columns).to(dtype)
            state['total'] = torch.empty_like(state['x'])
        state['weight'] = (1 + 0.2 * normal(columns)).to(dtype)
        state['codes'] = torch.empty((rows, columns), dtype=torch.int8, device='cuda')
        state['scales'] = torch.empty(rows, device='cuda')
        state['values'] = torch.empty_like(state['x'])
        return state
    if case['op'] == 'matmul':
        m, n, k = case['m'], case['n'], case['k']
        state['a'] = (normal(m, k) * 35).round().clamp(-127, 127).to(torch.int8)
        state['w'] = (normal(n, k) * 35).round().clamp(-127, 127).to(torch.int8)
        state['a_scales'] = 0.02 + 0.04 * torch.rand(m, device='cuda', generator=gen)
        state['w_scales'] = (0.5 + torch.rand(n, device='cuda', generator=gen)) / (35 * math.sqrt(k))
        state['bias'] = normal(n) if case['bias'] else None
        state['out'] = torch.empty((m, n), dtype=dtype, device='cuda')
        return state

    lengths, news = _lengths(case)
    pages, pool, row = _geometry(case)
    heads, kv_heads, head_size = case['heads'], case['kv_heads'], case['head_size']
    state['k'], state['k_scales'] = _pool(case, pool, gen)
    state['v'], state['v_scales'] = _pool(case, pool, gen)
    # the pages of a sequence lie anywhere in the pool
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in pages:
        table.append((order[at:at + n] + [0] * row)[:row])
        at += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    state['tokens'] = tokens = starts[-1]
    state['table'] = torch.tensor(table, dtype=torch.int32, device='cuda')
    state['lengths'] = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    state['starts'] = torch.tensor(starts, dtype=torch.int32, device='cuda')
    # queries, keys and values of a token lie side by side, as the joint projection leaves them
    width = (heads + 2 * kv_heads) * head_size
    state['joint'] = normal(tokens, width).to(dtype)
    state['new_k'] = state['joint'][:, heads * head_size:(heads + kv_heads) * head_size].unflatten(1, (kv_heads, head_size))
    state['new_v'] = state['joint'][:, (heads + kv_heads) * head_size:].unflatten(1, (kv_heads, head_size))
    state['q'] = state['joint'][:, :heads * head_size].unflatten(1, (heads, head_size))
    if case['op'] == 'append':
        state['k_values'] = torch.empty(state['k'].shape, dtype=dtype, device='cuda')
        state['v_values'] = torch.empty(state['v'].shape, dtype=dtype, device='cuda')
    else:
        state['out'] = torch.empty((tokens, heads, head_size), dtype=dtype, device='cuda')
        state['scale'] = 1 / math.sqrt(head_size)
    if own:
        from n2d2_b200 import runtime
        state['cache'] = runtime.KvCache(state['k'].data_ptr(), state['v'].data_ptr(), state['k_scales'].data_ptr(),
                                         state['v_scales'].data_ptr(), pool, kv_heads, case['page'], head_size)
        state['batch'] = runtime.KvBatch(len(lengths), state['table'].data_ptr(), row, state['lengths'].data_ptr(), tokens, case['new'],
                                         None if case['new'] == 1 else state['starts'].data_ptr())
    return state


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from n2d2_b200 import runtime
    case, stream = state['case'], state['stream']
    if case['op'] == 'norm':
        residual = case['residual']
        runtime.rmsnorm_quantize(state['x'].data_ptr(), case['rows'], case['columns'], state['weight'].data_ptr(), state['codes'].data_ptr(),
                                 state['scales'].data_ptr(), state['residual'].data_ptr() if residual else None,
                                 state['total'].data_ptr() if residual else None, dtype=case['dtype'], eps=1e-6, stream=stream)
        torch.mul(state['codes'], state['scales'][:, None], out=state['values'])
        return {'values': state['values'], 'scales': state['scales'], **({'total': state['total']} if residual else {})}
    if case['op'] == 'matmul':
        runtime.matmul_i8(state['a'].data_ptr(), state['a_scales'].data_ptr(), state['w'].data_ptr(), state['w_scales'].data_ptr(),
                          state['out'].data_ptr(), case['m'], case['n'], case['k'], dtype=case['dtype'],
                          bias=state['bias'].data_ptr() if case['bias'] else None, stream=stream)
        return state['out']
    if case['op'] == 'append':
        state['cache'].append(state['batch'], state['new_k'].data_ptr(), state['new_v'].data_ptr(), state['joint'].stride(0),
                              dtype=case['dtype'], stream=stream)
        torch.mul(state['k'], state['k_scales'][:, :, None, None], out=state['k_values'])
        torch.mul(state['v'], state['v_scales'][:, :, None, None], out=state['v_values'])
        return {'k': state['k_values'], 'v': state['v_values'], 'k_scales': state['k_scales'], 'v_scales': state['v_scales']}
    state['cache'].attention(state['batch'], state['q'].data_ptr(), state['out'].data_ptr(), case['heads'], state['scale'],
                             dtype=case['dtype'], q_stride=state['joint'].stride(0), window=case['window'], causal=case['causal'],
                             stream=stream)
    return state['out']


def _run_plain(state):
    case = state['case']
    dtype = TYPES[case['dtype']]
    if case['op'] == 'norm':
        h = state['x']
        if case['residual']:
            h = (h.float() + state['residual'].float()).to(dtype)
        wide = h.float()
        u = wide * state['weight'].float()
        step = u.abs().amax(1, keepdim=True) * (1 / 127)
        none = step <= TINY
        codes = (u * torch.where(none, 0.0, step.reciprocal())).round().clamp(-127, 127)
        scales = torch.where(none, 0.0, step) * torch.rsqrt(wide.square().mean(1, keepdim=True) + 1e-6)
        return {'values': (codes * scales).to(dtype), 'scales': scales[:, 0], **({'total': h} if case['residual'] else {})}
    if case['op'] == 'matmul':
        y = (state['a'].float() @ state['w'].float().T) * state['a_scales'][:, None] * state['w_scales']
        return (y if state['bias'] is None else y + state['bias']).to(dtype)
    if case['op'] == 'append':
        _plain_append(state, state['k'], state['k_scales'], state['new_k'])
        _plain_append(state, state['v'], state['v_scales'], state['new_v'])
        return {'k': (state['k'].float() * state['k_scales'][:, :, None, None]).to(dtype),
                'v': (state['v'].float() * state['v_scales'][:, :, None, None]).to(dtype),
                'k_scales': state['k_scales'], 'v_scales': state['v_scales']}
    return _plain_attention(state)


def _plain_append(state, pool, scales, x):
    """The pages that gain tokens, [sequence][page]: their old codes on the larger scale, the new tokens' beside them."""
    case = state['case']
    page = case['page']
    end = state['lengths'][:, None].long()
    new = (state['starts'][1:] - state['starts'][:-1])[:, None].long()
    begin = (end - new).clamp(min=0)
    touched = begin // page + torch.arange((case['new'] + page - 2) // page + 1, device='cuda')
    touched = torch.minimum(touched, ((end - 1) // page).clamp(min=0))     # the last one may stand there more than once, the same each time
    pages = torch.gather(state['table'].long(), 1, touched)
    place = touched[:, :, None] * page + torch.arange(page, device='cuda')
    fresh = (place >= begin[:, :, None]) & (place < end[:, :, None])
    old = place < begin[:, :, None]
    token = (state['starts'][:-1].long()[:, None, None] + place - (end - new)[:, :, None]).clamp(0, state['tokens'] - 1)
    values = x[token].float().transpose(2, 3)                               # [sequence][page][head][place][head_size]
    fresh, old = fresh[:, :, None, :, None], old[:, :, None, :, None]
    step = (values.abs() * fresh).amax((3, 4)) * (1 / 127)
    held = scales[pages]
    before = torch.where(old[..., 0].any(3), held, 0.0)
    after = torch.maximum(before, torch.where(step <= TINY, 0.0, step))
    ratio = torch.where(after > 0, before / after, 0.0)[..., None, None]
    inverse = torch.where(after > 0, after.reciprocal(), 0.0)[..., None, None]
    codes = pool[pages]
    moved = (codes.float() * ratio).round()
    taken = (values * inverse).round().clamp(-127, 127)
    pool[pages] = torch.where(fresh, taken, torch.where(old, moved, codes.float())).to(torch.int8)
    scales[pages] = torch.where(fresh.any(3)[..., 0], after, held)


def _plain_attention(state):
    case = state['case']
    batch, new, heads, kv_heads, size, page = (case[k] for k in ('batch', 'new', 'heads', 'kv_heads', 'head_size', 'page'))
    starts, lengths = state['starts'].long(), state['lengths'].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(new, device='cuda')
    token = (starts[:-1, None] + i).clamp(max=state['tokens'] - 1)
    q = state['q'][token].float().unflatten(2, (kv_heads, heads // kv_heads)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    pages = state['table'].long()
    keys = pages.shape[1] * page

    def cached(codes, scales):
        x = codes[pages].float() * scales[pages][..., None, None]           # [batch][page][head][place][size]
        return x.permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, keys, size)

    scores = (q @ cached(state['k'], state['k_scales']).transpose(2, 3)) * state['scale']
    j = torch.arange(keys, device='cuda')
    position = (lengths - count)[:, None] + i
    visible = (j < lengths[:, None, None]).expand(batch, new, keys)
    if case['causal']:
        visible = visible & (j <= position[:, :, None])
        if case['window']:
            visible = visible & (j > position[:, :, None] - case['window'])
    scores = scores.unflatten(2, (heads // kv_heads, new))
    scores.masked_fill_(~visible[:, None, None], -math.inf)
    largest = scores.amax(4, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = scores.sub_(largest).exp_()
    total = p.sum(4).flatten(2, 3)[..., None]
    out = (p.flatten(2, 3) @ cached(state['v'], state['v_scales'])) / total
    out = torch.where(total > 0, out, 0.0).unflatten(2, (heads // kv_heads, new)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    t = torch.arange(state['tokens'], device='cuda')
    sequence = torch.searchsorted(starts[1:], t, right=True)
    return out[sequence, t - starts[sequence]].to(TYPES[case['dtype']])


def work(case):
    """Inputs read once, outputs written once; 2 operations per multiply-accumulate of the products."""
    item = {'f32': 4, 'f16': 2, 'bf16': 2}[case['dtype']]
    if case['op'] == 'norm':
        n = case['rows'] * case['columns']
        return {'bytes': n * (item * (3 if case['residual'] else 1) + 1) + item * case['columns'] + 4 * case['rows'], 'flops': 6 * n}
    if case['op'] == 'matmul':
        m, n, k = case['m'], case['n'], case['k']
        return {'bytes': m * k + n * k + 4 * (m + n) + (4 * n if case['bias'] else 0) + m * n * item, 'flops': 2 * m * n * k}
    lengths, news = _lengths(case)
    heads, kv_heads, size = case['heads'], case['kv_heads'], case['head_size']
    if case['op'] == 'append':
        # the new tokens' values in and their codes out (keys and values), the page of the last old token both ways
        n = sum(news[b] for b in range(len(news)) if lengths[b]) * kv_heads * size
        return {'bytes': 2 * n * (item + 1), 'flops': 4 * n}
    pairs = cached = 0
    for end, new in zip(lengths, news):
        if not end:
            continue
        window = case['window'] or end
        if not case['causal']:
            pairs, cached = pairs + new * end, cached + end
            continue
        # query at position p sees min(p + 1, window) tokens
        first = end - new
        full = max(0, min(new, end - max(first, window - 1)))
        short = new - full
        pairs += full * window + short * first + short * (short + 1) // 2
        cached += end - max(0, first - window + 1)
    scales = 8 * kv_heads * (cached // case['page'])
    return {'bytes': 2 * cached * kv_heads * size + scales + 2 * sum(news) * heads * size * item, 'flops': 4 * pairs * heads * size}


def exact(case, seed):
    state = prepare(case, seed)
    f64 = torch.float64
    if case['op'] == 'norm':
        h = state['x']
        if case['residual']:
            # the norm is taken of the sum as it is stored
            total = h.to(f64) + state['residual'].to(f64)
            h = total.to(TYPES[case['dtype']])
        values, scales = torch.empty(h.shape, dtype=f64, device='cuda'), torch.empty(h.shape[0], dtype=f64, device='cuda')
        for at in range(0, h.shape[0], 512):
            rows = h[at:at + 512].to(f64)
            u = rows * state['weight'].to(f64)
            step = u.abs().max(1).values / 127
            scales[at:at + 512] = step / torch.sqrt((rows * rows).sum(1) / rows.shape[1] + 1e-6)
            codes = torch.round(u / step[:, None]).nan_to_num(0.0)
            values[at:at + 512] = codes * scales[at:at + 512, None]
        return {'values': values, 'scales': scales, **({'total': total} if case['residual'] else {})}
    if case['op'] == 'matmul':
        y = torch.mm(state['a'].to(f64), state['w'].to(f64).t())
        y = y * torch.outer(state['a_scales'].to(f64), state['w_scales'].to(f64))
        return y + state['bias'].to(f64) if case['bias'] else y
    lengths, news = _lengths(case)
    table = state['table'].cpu()
    page = case['page']
    out, at = {}, 0
    if case['op'] == 'append':
        for name, new in (('k', state['new_k']), ('v', state['new_v'])):
            codes, scales, at = state[name].to(f64), state[name + '_scales'].to(f64), 0
            for b, (end, n) in enumerate(zip(lengths, news)):
                begin = end - n
                for p in range(max(begin, 0) // page, -(-end // page)):
                    lo, hi, number = max(begin, p * page), min(end, (p + 1) * page), int(table[b, p])
                    x = new[at + lo - begin:at + hi - begin].to(f64).transpose(0, 1)
                    held = scales[number] if lo > p * page else torch.zeros_like(scales[number])
                    grown = torch.maximum(held, x.abs().amax((1, 2)) / 127)
                    old = codes[number, :, :lo - p * page]
                    codes[number, :, :lo - p * page] = torch.round(old * (held / grown)[:, None, None])
                    codes[number, :, lo - p * page:hi - p * page] = torch.round(x / grown[:, None, None])
                    scales[number] = grown
                at += n
            out[name], out[name + '_scales'] = codes * scales[:, :, None, None], scales
        return out
    heads, kv_heads, size = case['heads'], case['kv_heads'], case['head_size']
    result = torch.zeros(state['tokens'], heads, size, dtype=f64, device='cuda')
    for b, (end, n) in enumerate(zip(lengths, news)):
        if end:
            used = table[b, :-(-end // page)].long().cuda()
            position = torch.arange(end - n, end, device='cuda')[:, None]
            j = torch.arange(end, device='cuda')[None]
            hidden = torch.zeros((n, end), dtype=torch.bool, device='cuda')
            if case['causal']:
                hidden = j > position
                if case['window']:
                    hidden = hidden | (j <= position - case['window'])
            for h in range(heads):
                g = h // (heads // kv_heads)
                k = (state['k'][used, g].to(f64) * state['k_scales'][used, g].to(f64)[:, None, None]).flatten(0, 1)[:end]
                v = (state['v'][used, g].to(f64) * state['v_scales'][used, g].to(f64)[:, None, None]).flatten(0, 1)[:end]
                s = state['q'][at:at + n, h].to(f64) @ k.t() * state['scale']
                result[at:at + n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
        at += n
    return result
