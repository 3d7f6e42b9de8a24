"""What the operators around the MoE layer are measured on: embedding lookup and its gradient, the global gradient norm with
clipping, and low-rank adapters beside a shared projection.

Every operator has a plain form here (elementary torch operations in 32 bits) and the call of the library's own kernels
(`own`). A case is a dict of plain values; `kind` names the operator:

* `lookup`       rows of a table by index, scaled; indices outside the table (negative = masked) give zero rows
* `embed_grad`   gradient of the lookup, dense, in the table's type
* `embed_accum`  the same, added to an fp32 buffer that the training loop keeps
* `norm`         L2 norm over a list of gradient tensors
* `clip`         clipping by that norm in place (`reached` false: the usual step, in which nothing has to be scaled) or from
                 fp32 accumulators into bf16 gradients
* `lora`         y = x W^T + scaling[e] (x A_e^T) B_e^T, e the adapter of the row (negative = none)
* `lora_train`   the same, with the gradients of x, A and B
"""
import math

import torch

own = False

_TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed():
    return [
        # one decoded token of one sequence: pure latency
        {'name': 'lookup_one_token', 'kind': 'lookup', 'tokens': 1, 'rows': 32768, 'hidden': 7168, 'type': 'bf16', 'masked': 0.0},
        # a prefill batch at the layer's hidden size, padded positions masked
        {'name': 'lookup_prefill', 'kind': 'lookup', 'tokens': 16384, 'rows': 131072, 'hidden': 7168, 'type': 'bf16', 'masked': 0.05},
        # n-gram memory entries stored in 8 bits with one scale per 128 columns
        {'name': 'lookup_fp8_entries', 'kind': 'lookup', 'tokens': 32760, 'rows': 262144, 'hidden': 1024, 'type': 'e4m3', 'masked': 0.1},
        # training step of a large batch: dense gradient of the table, frequent tokens repeat
        {'name': 'embed_grad_batch', 'kind': 'embed_grad', 'tokens': 16384, 'rows': 65536, 'hidden': 7168, 'type': 'bf16', 'masked': 0.02},
        # ragged micro-batch into a persistent fp32 buffer, odd width and vocabulary
        {'name': 'embed_accum_ragged', 'kind': 'embed_accum', 'tokens': 5001, 'rows': 50001, 'hidden': 1003, 'type': 'fp16', 'masked': 0.0},
        # many small gradients (norms, biases, adapters): launch and bookkeeping count
        {'name': 'norm_small_tensors', 'kind': 'norm', 'tensors': 240, 'numel': 50000, 'type': 'bf16'},
        # the usual step: the norm stays below the limit, expert gradients are only read
        {'name': 'clip_experts_below_limit', 'kind': 'clip', 'tensors': 24, 'numel': 24000000, 'type': 'bf16', 'reached': False},
        # fp32 accumulators -> clipped bf16 gradients
        {'name': 'clip_fp32_to_bf16', 'kind': 'clip', 'tensors': 40, 'numel': 8000000, 'type': 'fp32', 'reached': True},
        # one token through the shared expert's first projection
        {'name': 'lora_one_token', 'kind': 'lora', 'tokens': 1, 'k': 7168, 'n': 4096, 'rank': 16, 'adapters': 4, 'none': 0.0, 'order': 'mixed'},
        # decode: every row another request, many adapters at once
        {'name': 'lora_decode_many_adapters', 'kind': 'lora', 'tokens': 96, 'k': 7168, 'n': 4096, 'rank': 16, 'adapters': 64, 'none': 0.1,
         'order': 'mixed'},
        # prefill: a few long ragged requests, one of them without an adapter
        {'name': 'lora_prefill_ragged', 'kind': 'lora', 'tokens': 8101, 'k': 7168, 'n': 4096, 'rank': 64, 'adapters': 6, 'none': 0.1,
         'order': 'requests'},
        # fine-tuning several adapters of one base model in one batch
        {'name': 'lora_train_step', 'kind': 'lora_train', 'tokens': 4099, 'k': 7168, 'n': 4096, 'rank': 32, 'adapters': 4, 'none': 0.0,
         'order': 'requests'},
    ]


def _spread(rng, low, high):
    """A whole number between both ends, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(['lookup', 'embed_grad', 'embed_accum', 'norm', 'clip', 'lora', 'lora_train'])
    if kind == 'lookup':
        kind_type = rng.choice(['bf16', 'fp16', 'fp32', 'e4m3'])
        hidden = 128 * rng.randint(1, 56) if kind_type == 'e4m3' else rng.choice([_spread(rng, 64, 7168), 8 * rng.randint(8, 896)])
        return {'kind': kind, 'tokens': _spread(rng, 1, 8192 if kind_type == 'fp32' else 16384), 'rows': _spread(rng, 1000, 131072), 'hidden': hidden,
                'type': kind_type, 'masked': rng.choice([0.0, 0.02, 0.5])}
    if kind in ('embed_grad', 'embed_accum'):
        return {'kind': kind, 'tokens': _spread(rng, 1, 16384), 'rows': _spread(rng, 1000, 32000),
                'hidden': rng.choice([_spread(rng, 64, 4096), 8 * rng.randint(8, 512)]), 'type': rng.choice(['bf16', 'fp16', 'fp32']),
                'masked': rng.choice([0.0, 0.02, 0.5])}
    if kind == 'norm':
        tensors = _spread(rng, 1, 400)
        return {'kind': kind, 'tensors': tensors, 'numel': _spread(rng, 100, min(20000000, 200000000 // tensors)),
                'type': rng.choice(['bf16', 'fp16', 'fp32'])}
    if kind == 'clip':
        tensors = _spread(rng, 1, 200)
        reached = rng.random() < 0.5
        return {'kind': kind, 'tensors': tensors, 'numel': _spread(rng, 100, min(20000000, 200000000 // tensors)),
                'type': 'fp32' if reached else rng.choice(['bf16', 'fp16', 'fp32']), 'reached': reached}
    tokens = _spread(rng, 1, 8101 if kind == 'lora' else 4099)
    return {'kind': kind, 'tokens': tokens, 'k': 8 * _spread(rng, 32, 896), 'n': 8 * _spread(rng, 32, 512),
            'rank': rng.choice([8, 16, 32, 64]), 'adapters': _spread(rng, 1, 64 if tokens <= 512 and kind == 'lora' else 8),
            'none': rng.choice([0.0, 0.1]), 'order': 'mixed' if tokens <= 256 else rng.choice(['requests', 'requests', 'mixed'])}


def _scale(case):
    return math.sqrt(case['hidden'])


def _sizes(case):
    """Element counts of the tensors of a gradient list: ragged around `numel`, one of them a hundredth of it."""
    numel, count = case['numel'], case['tensors']
    return [max(1, numel // 100) if i % 7 == 3 else max(1, numel - (i * 37) % max(1, numel // 3)) for i in range(count)]


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _ids(tokens, rows, masked, gen):
    """Token ids with a few very frequent ones, a share of them masked (-1)."""
    u = torch.rand(tokens, device='cuda', generator=gen, dtype=torch.float64)
    ids = (rows ** u - 1).long().clamp_(0, rows - 1)          # density ~ 1 / (1 + id)
    ids = (ids * 7919) % rows                                 # frequent ids lie anywhere in the table
    hide = torch.rand(tokens, device='cuda', generator=gen) < masked
    return torch.where(hide, torch.full_like(ids, -1), ids)


def prepare(case, seed):
    gen, kind = _gen(seed), case['kind']
    randn = lambda *shape: torch.randn(*shape, device='cuda', generator=gen)      # noqa: E731
    state = {'case': dict(case)}
    if kind == 'lookup':
        rows, hidden = case['rows'], case['hidden']
        state['ids'] = _ids(case['tokens'], rows, case['masked'], gen)
        if case['type'] == 'e4m3':
            state['table'] = (randn(rows, hidden) * 64).clamp_(-448, 448).to(torch.float8_e4m3fn)
            state['sf'] = torch.rand(rows, hidden // 128, device='cuda', generator=gen) * 0.01 + 1e-4
        else:
            state['table'] = torch.randn(rows, hidden, device='cuda', generator=gen, dtype=_TYPES[case['type']]) * 0.02
            state['sf'] = None
    elif kind in ('embed_grad', 'embed_accum'):
        state['ids'] = _ids(case['tokens'], case['rows'], case['masked'], gen)
        state['dy'] = (randn(case['tokens'], case['hidden']) * 0.01).to(_TYPES[case['type']])
        if kind == 'embed_grad':
            state['rows'] = case['rows']
        else:
            state['acc'] = randn(case['rows'], case['hidden']) * 0.01
    elif kind in ('norm', 'clip'):
        dtype = _TYPES[case['type']]
        sizes = _sizes(case)
        # gradients lie one after the other in one buffer, as a bucket holds them; odd sizes leave odd offsets
        flat = torch.randn(sum(sizes), device='cuda', generator=gen, dtype=dtype) * 1e-3
        state['grads'] = list(flat.split(sizes))
        if kind == 'clip':
            norm = 1e-3 * math.sqrt(sum(sizes))
            state['max_norm'] = norm * 0.25 if case['reached'] else norm * 64
            # what comes back is the whole buffer that the clipped gradients lie in
            state['flat'] = torch.empty(sum(sizes), device='cuda', dtype=torch.bfloat16) if case['reached'] else flat
            state['out'] = list(state['flat'].split(sizes)) if case['reached'] else None
    else:
        tokens, k, n, r, e = (case[x] for x in ('tokens', 'k', 'n', 'rank', 'adapters'))
        bf16 = torch.bfloat16
        state['x'] = randn(tokens, k).to(bf16)
        state['w'] = (randn(n, k) * k ** -0.5).to(bf16)
        state['a'] = (randn(e, r, k) * k ** -0.5).to(bf16)
        state['b'] = (randn(e, n, r) * r ** -0.5).to(bf16)
        state['scaling'] = torch.rand(e, device='cuda', generator=gen) + 0.5
        idx = torch.randint(0, e, (tokens,), device='cuda', generator=gen)
        idx = torch.where(torch.rand(tokens, device='cuda', generator=gen) < case['none'], torch.full_like(idx, -1), idx)
        if case['order'] == 'requests':
            # the tokens of a request lie together: ragged runs, the number of rows per adapter as drawn
            idx = idx.sort().values
        state['idx'] = idx.to(torch.int32)
        if kind == 'lora_train':
            state['dy'] = randn(tokens, n).to(bf16)
            for name in ('x', 'a', 'b'):
                state[name].requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_lookup(s):
    table, ids, scale = s['table'], s['ids'], _scale(s['case'])
    valid = (ids >= 0) & (ids < table.size(0))
    inside = ids.clamp(0, table.size(0) - 1)
    # (8-bit types are picked as bytes: not every torch indexing kernel knows them)
    rows = (table[inside] if s['sf'] is None else table.view(torch.uint8)[inside].view(table.dtype)).float()
    if s['sf'] is not None:
        sf = s['sf'][inside]
        rows = (rows.view(rows.size(0), -1, 128) * sf.unsqueeze(-1)).view(rows.shape)
    rows = torch.where(valid.unsqueeze(1), rows * scale, torch.zeros((), device=rows.device))
    return rows.to(torch.bfloat16 if s['sf'] is not None else table.dtype)


def _plain_embed_sum(ids, dy, rows, scale):
    valid = (ids >= 0) & (ids < rows)
    contribution = torch.where(valid.unsqueeze(1), dy.float(), torch.zeros((), device=dy.device))
    return torch.zeros(rows, dy.size(1), device=dy.device).index_add_(0, ids.clamp(0, rows - 1), contribution) * scale


def _plain_norm(grads):
    return torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()


def _plain_clip(s):
    norm = _plain_norm(s['grads'])
    factor = (s['max_norm'] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * factor) for o, g in zip(s['out'] or s['grads'], s['grads'])]
    return [norm, s['flat']]


def _plain_lora_parts(s):
    """fp32 operands and the rows' adapters as a scaled one-hot matrix [tokens, adapters]."""
    e = s['a'].size(0)
    hot = (s['idx'].unsqueeze(1) == torch.arange(e, device=s['idx'].device)).float() * s['scaling']
    return s['x'].detach().float(), s['w'].float(), s['a'].detach().float(), s['b'].detach().float(), hot


def _plain_lora(s):
    x, w, a, b, hot = _plain_lora_parts(s)
    e, r, k = a.shape
    t = (x @ a.view(e * r, k).t()).view(-1, e, r) * hot.unsqueeze(-1)
    return (x @ w.t() + t.flatten(1) @ b.transpose(1, 2).reshape(e * r, -1)).to(s['x'].dtype)


def _plain_lora_train(s):
    x, w, a, b, hot = _plain_lora_parts(s)
    e, r, k = a.shape
    dy = s['dy'].float()
    t = (x @ a.view(e * r, k).t()).view(-1, e, r) * hot.unsqueeze(-1)
    b_all = b.transpose(1, 2).reshape(e * r, -1)
    y = x @ w.t() + t.flatten(1) @ b_all
    dt = ((dy @ b_all.t()).view(-1, e, r) * hot.unsqueeze(-1)).flatten(1)
    dx = dy @ w + dt @ a.view(e * r, k)
    da = (dt.t() @ x).view(e, r, k)
    db = (dy.t() @ t.flatten(1)).view(-1, e, r).permute(1, 0, 2)
    return [v.to(s['x'].dtype) for v in (y, dx, da, db)]


# ------------------------------------------------------------------------------------------------ the library's calls
def _own(s):
    kind = s['case']['kind']
    if kind in ('lookup', 'embed_grad', 'embed_accum'):
        from deep_ep.ops.embedding import embedding_grad, embedding_lookup
        scale = _scale(s['case'])
        if kind == 'lookup':
            return embedding_lookup(s['table'], s['ids'], scale, table_sf=s['sf'])
        if kind == 'embed_grad':
            return embedding_grad(s['dy'], s['ids'], s['rows'], scale)
        return embedding_grad(s['dy'], s['ids'], s['acc'].size(0), scale, out=s['acc'], accumulate=True)
    if kind in ('norm', 'clip'):
        from deep_ep.ops.grad_norm import clip_grad_norm_, grad_norm
        if kind == 'norm':
            return grad_norm(s['grads'])
        norm = clip_grad_norm_(s['grads'], s['max_norm'], out=s['out'])
        return [norm, s['flat']]
    from deep_ep.ops.lora import lora_linear
    y = lora_linear(s['x'], s['w'], s['a'], s['b'], s['idx'], s['scaling'])
    if kind == 'lora':
        return y
    return [y.detach(), *torch.autograd.grad(y, (s['x'], s['a'], s['b']), s['dy'])]


def run(state):
    if own:
        return _own(state)
    kind = state['case']['kind']
    if kind == 'lookup':
        return _plain_lookup(state)
    if kind == 'embed_grad':
        return _plain_embed_sum(state['ids'], state['dy'], state['rows'], _scale(state['case'])).to(state['dy'].dtype)
    if kind == 'embed_accum':
        return state['acc'].add_(_plain_embed_sum(state['ids'], state['dy'], state['acc'].size(0), _scale(state['case'])))
    if kind == 'norm':
        return _plain_norm(state['grads'])
    if kind == 'clip':
        return _plain_clip(state)
    return _plain_lora(state) if kind == 'lora' else _plain_lora_train(state)


# ------------------------------------------------------------------------------------------------ the work of one pass
def work(case):
    kind = case['kind']
    size = {'bf16': 2, 'fp16': 2, 'fp32': 4, 'e4m3': 1}
    if kind == 'lookup':
        t, h = case['tokens'], case['hidden']
        live = t * (1 - case['masked'])
        # rows that occur again need not be read again
        distinct = min(live, _distinct(live, case['rows']))
        row = h * size[case['type']] + (h // 128 * 4 if case['type'] == 'e4m3' else 0)
        out = h * (2 if case['type'] == 'e4m3' else size[case['type']])
        return {'bytes': int(8 * t + distinct * row + t * out), 'flops': int(live * h)}
    if kind in ('embed_grad', 'embed_accum'):
        t, h, v = case['tokens'], case['hidden'], case['rows']
        live = t * (1 - case['masked'])
        read = 8 * t + live * h * size[case['type']]
        written = v * h * size[case['type']] if kind == 'embed_grad' else 2 * min(live, _distinct(live, v)) * h * 4
        return {'bytes': int(read + written), 'flops': int(2 * live * h)}
    if kind in ('norm', 'clip'):
        total = sum(_sizes(case))
        written = total * 2 if kind == 'clip' and case['reached'] else 0
        return {'bytes': total * size[case['type']] + written, 'flops': total * (3 if written else 2)}
    t, k, n, r = case['tokens'], case['k'], case['n'], case['rank']
    e = min(case['adapters'], t)
    operands = 2 * (t * k + n * k + t * n + e * r * (k + n)) + 4 * t
    flops = 2 * t * k * n + 2 * t * r * (k + n)
    if kind == 'lora_train':
        # dx needs W again in another order of summation but not from memory; dy in, dx, dA and dB out
        return {'bytes': operands + 2 * (t * n + t * k + case['adapters'] * r * (k + n)), 'flops': 2 * flops + 2 * t * r * (k + n)}
    return {'bytes': operands, 'flops': flops}


def _distinct(live, rows):
    """About how many different ids `_ids` gives: the sum over ids of 1 - (1 - p)^live with p ~ 1 / ((1 + id) ln rows)."""
    total, lo = 0.0, 1.0
    while lo < rows:
        hi = min(lo * 1.25, rows)
        p = math.log((1 + hi) / (1 + lo)) / math.log(rows) / max(hi - lo, 1e-9)
        total += (hi - lo) * (1 - math.exp(-live * p))
        lo = hi
    return max(1.0, total)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind, f64 = case['kind'], torch.float64
    if kind == 'lookup':
        out = torch.zeros(case['tokens'], case['hidden'], device='cuda', dtype=f64)
        live = torch.nonzero(s['ids'] >= 0).flatten()
        picked = s['table'].view(torch.uint8)[s['ids'][live]].view(torch.float8_e4m3fn) if s['sf'] is not None else s['table'][s['ids'][live]]
        picked = picked.to(f64)
        if s['sf'] is not None:
            picked = picked * torch.repeat_interleave(s['sf'][s['ids'][live]].to(f64), 128, dim=1)
        out[live] = picked * math.sqrt(case['hidden'])
        return out
    if kind in ('embed_grad', 'embed_accum'):
        live = torch.nonzero(s['ids'] >= 0).flatten()
        # sums by sorted id through running totals of each run
        order = live[torch.argsort(s['ids'][live])]
        ids, where = torch.unique_consecutive(s['ids'][order], return_inverse=True)
        sums = torch.zeros(ids.numel(), case['hidden'], device='cuda', dtype=f64)
        for c in range(0, order.numel(), 4096):
            sums.index_add_(0, where[c:c + 4096], s['dy'][order[c:c + 4096]].to(f64))
        out = torch.zeros(case['rows'], case['hidden'], device='cuda', dtype=f64) if kind == 'embed_grad' else s['acc'].to(f64)
        out[ids] += sums * math.sqrt(case['hidden'])
        return out
    if kind in ('norm', 'clip'):
        total = math.fsum(float(torch.linalg.vector_norm(g, dtype=f64)) ** 2 for g in s['grads'])
        norm = math.sqrt(total)
        head = torch.tensor(norm, device='cuda', dtype=f64)
        if kind == 'norm':
            return head
        factor = min(1.0, s['max_norm'] / (norm + 1e-6))
        return [head, torch.cat([g.to(f64) * factor for g in s['grads']])]
    x, w, a, b = (s[name].detach().to(f64) for name in ('x', 'w', 'a', 'b'))
    y = x @ w.t()
    groups = [(e, torch.nonzero(s['idx'] == e).flatten(), float(s['scaling'][e])) for e in range(case['adapters'])]
    for e, rows, scale in groups:
        y[rows] += scale * ((x[rows] @ a[e].t()) @ b[e].t())
    if kind == 'lora':
        return y
    dy = s['dy'].to(f64)
    dx, da, db = dy @ w, torch.zeros_like(a), torch.zeros_like(b)
    for e, rows, scale in groups:
        back = scale * (dy[rows] @ b[e])
        dx[rows] += back @ a[e]
        da[e] = back.t() @ x[rows]
        db[e] = scale * (dy[rows].t() @ (x[rows] @ a[e].t()))
    return [y, dx, da, db]
