"""
Cases of the expert-layer operators and their plain forms.

Four operators of a mixture-of-experts feed-forward layer, as a program that serves such a layer meets them:

* ``route``    the router: the k best experts of every token, their gates, and the plan that sorts the (token, expert)
               pairs by expert;
* ``grouped``  the experts' matrix products over that plan: one ragged product per expert, bfloat16, float16, float32 or
               8-bit integers with scales, rows gathered by index, optionally with the gated activation;
* ``int8``     a dense product in 8-bit integers: tokens quantised with a scale each, weights with a scale per channel;
* ``combine``  the gate-weighted sum of every token's expert rows.

``run`` computes the plain form in elementary torch operations while ``own`` is false, and calls the framework's
operators where it is true.  Sizes are generic, from a single token to a long prompt; some come from this repository's
convolution layers (288 -> 768 channels), which are products of the same kind.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # routing: one decoding step of a few sequences; a long prompt batch whose padding tokens have every expert masked
        {'name': 'route_step', 'op': 'route', 'tokens': 4, 'experts': 64, 'k': 8, 'dtype': 'fp32', 'padded': 0.0},
        {'name': 'route_prompt', 'op': 'route', 'tokens': 16384, 'experts': 128, 'k': 8, 'dtype': 'bf16', 'padded': 0.06},
        # up and gate products of four decoding sequences: 32 rows over 64 experts, bound by the weights they read
        {'name': 'grouped_step', 'op': 'grouped', 'tokens': 4, 'k': 8, 'experts': 64, 'inner': 2048, 'outer': 1280,
         'dtype': 'bf16', 'gather': True, 'gated': True, 'act': 'silu', 'bias': False, 'skew': 0.0},
        # the same layer on a prompt of 4096 tokens, experts unevenly loaded: bound by the tensor cores
        {'name': 'grouped_prompt', 'op': 'grouped', 'tokens': 4096, 'k': 8, 'experts': 64, 'inner': 2048, 'outer': 1280,
         'dtype': 'bf16', 'gather': True, 'gated': True, 'act': 'silu', 'bias': False, 'skew': 0.7},
        # down product of a medium batch: rows already sorted, odd counts, a few experts without rows
        {'name': 'grouped_down', 'op': 'grouped', 'tokens': 389, 'k': 4, 'experts': 32, 'inner': 1408, 'outer': 2048,
         'dtype': 'fp16', 'gather': False, 'gated': False, 'act': 'identity', 'bias': True, 'skew': 1.0},
        # float32, the runtime's default storage, with an odd row length; channel counts of an Inception module
        {'name': 'grouped_float', 'op': 'grouped', 'tokens': 777, 'k': 2, 'experts': 8, 'inner': 289, 'outer': 768,
         'dtype': 'fp32', 'gather': True, 'gated': False, 'act': 'relu', 'bias': True, 'skew': 0.5},
        # quantised experts: rows and weights in 8-bit integers with their scales
        {'name': 'grouped_int8', 'op': 'grouped', 'tokens': 2048, 'k': 4, 'experts': 32, 'inner': 1280, 'outer': 2048,
         'dtype': 'int8', 'gather': False, 'gated': False, 'act': 'identity', 'bias': False, 'skew': 0.7},
        # dense 8-bit products with the tokens quantised on the way in: one token, an odd batch, a long prompt
        {'name': 'int8_token', 'op': 'int8', 'tokens': 1, 'inner': 4096, 'outer': 8192, 'dtype': 'bf16', 'bias': False,
         'act': 'identity'},
        {'name': 'int8_batch', 'op': 'int8', 'tokens': 133, 'inner': 2048, 'outer': 5003, 'dtype': 'fp16', 'bias': True,
         'act': 'relu'},
        {'name': 'int8_prompt', 'op': 'int8', 'tokens': 8192, 'inner': 4096, 'outer': 8192, 'dtype': 'bf16', 'bias': False,
         'act': 'identity'},
        # the weighted sum at the end of the layer: a decoding step; a long prompt with padding tokens
        {'name': 'combine_step', 'op': 'combine', 'tokens': 4, 'k': 8, 'channels': 2048, 'dtype': 'bf16', 'padded': 0.0},
        {'name': 'combine_prompt', 'op': 'combine', 'tokens': 8192, 'k': 8, 'channels': 2048, 'dtype': 'fp16',
         'padded': 0.06},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _length(rng, low, high):
    """A row length: mostly a multiple of 64 as layers have it, sometimes any number (rows that start at odd addresses)."""
    n = _log_uniform(rng, low, high)
    return n if rng.random() < 0.25 else max(low, n // 64 * 64)


def draw(rng):
    op = rng.choice(('route', 'grouped', 'grouped', 'int8', 'int8', 'combine'))
    if op == 'route':
        experts = _log_uniform(rng, 4, 256)
        return {'op': op, 'tokens': _log_uniform(rng, 1, 16384), 'experts': experts,
                'k': rng.randint(1, min(8, experts)), 'dtype': rng.choice(('bf16', 'fp16', 'fp32')),
                'padded': rng.choice((0.0, 0.0, 0.1))}
    if op == 'grouped':
        dtype = rng.choice(('bf16', 'bf16', 'fp16', 'int8', 'fp32'))
        case = {'op': op, 'tokens': _log_uniform(rng, 1, 2048), 'k': rng.randint(1, 4), 'experts': _log_uniform(rng, 4, 64),
                'inner': _length(rng, 64, 2048), 'outer': _length(rng, 64, 2048 if dtype != 'fp32' else 1024), 'dtype': dtype,
                'gather': rng.random() < 0.5, 'gated': rng.random() < 0.4, 'act': rng.choice(('identity', 'relu', 'silu')),
                'bias': rng.random() < 0.5, 'skew': round(rng.uniform(0.0, 1.0), 2)}
        return case
    if op == 'int8':
        return {'op': op, 'tokens': _log_uniform(rng, 1, 4096), 'inner': _length(rng, 64, 4096),
                'outer': _length(rng, 64, 8192), 'dtype': rng.choice(('bf16', 'fp16', 'fp32')), 'bias': rng.random() < 0.5,
                'act': rng.choice(('identity', 'relu', 'silu'))}
    return {'op': op, 'tokens': _log_uniform(rng, 1, 8192), 'k': rng.randint(1, 8), 'channels': _length(rng, 64, 2048),
            'dtype': rng.choice(('bf16', 'fp16', 'fp32')), 'padded': rng.choice((0.0, 0.1))}


def _loads(case):
    """Rows per expert of a grouped case, heaviest first: shares fall as rank^-skew; part of the case, not of the seed."""
    rows, experts = case['tokens'] * case['k'], case['experts']
    pick = random.Random(f"{rows} {experts} {case['skew']}")
    shares = [(i + 1.0) ** -case['skew'] for i in range(experts)]
    counts = [0] * experts
    for e in pick.choices(range(experts), weights=shares, k=rows):
        counts[e] += 1
    return counts


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _activations(gen, shape):
    """Hidden states: unit variance with a few channels an order of magnitude larger, as layers after a norm have them."""
    x = torch.randn(shape, generator=gen, device='cuda')
    loud = torch.rand(shape[-1], generator=gen, device='cuda') < 0.01
    return x * (1.0 + 9.0 * loud)


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    op, state = case['op'], {'case': case}
    if op == 'route':
        logits = 1.5 * torch.randn(case['tokens'], case['experts'], generator=gen, device='cuda')
        logits += torch.randn(case['experts'], generator=gen, device='cuda')            # experts the router prefers
        pad = torch.rand(case['tokens'], generator=gen, device='cuda') < case['padded']
        logits[pad] = -math.inf
        state['logits'] = logits.to(DTYPES[case['dtype']])
        return state
    if op == 'grouped':
        counts = torch.tensor(_loads(case), device='cuda')
        order = torch.randperm(case['experts'], generator=gen, device='cuda')
        counts = counts[order]
        rows_total = case['tokens'] * case['k']
        state['widest'] = max(_loads(case))
        state['offsets'] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        shape_w = (case['experts'], case['outer'] * (2 if case['gated'] else 1), case['inner'])
        x = _activations(gen, (case['tokens'] if case['gather'] else rows_total, case['inner']))
        state['rows'] = None
        if case['gather']:
            shuffled = torch.randperm(rows_total, generator=gen, device='cuda')
            state['rows'] = (shuffled // case['k']).to(torch.int32)
        state['row_scale'] = state['channel_scale'] = state['bias'] = None
        if case['dtype'] == 'int8':
            # quantised once, before the layer runs: whole rows to [-127, 127] by their largest magnitude
            state['x'] = (x * (127.0 / x.abs().amax(1, keepdim=True))).round().to(torch.int8)
            state['row_scale'] = (x.abs().amax(1) / 127.0)
            state['weight'] = torch.randint(-127, 128, shape_w, generator=gen, device='cuda', dtype=torch.int8)
            state['channel_scale'] = (0.5 + torch.rand(shape_w[:2], generator=gen, device='cuda')) / (73.0 * math.sqrt(case['inner']))
        else:
            dtype = DTYPES[case['dtype']]
            state['x'] = x.to(dtype)
            state['weight'] = torch.empty(shape_w, dtype=dtype, device='cuda').normal_(0.0, case['inner'] ** -0.5, generator=gen)
        if case['bias']:
            state['bias'] = 0.1 * torch.randn(shape_w[:2], generator=gen, device='cuda')
        return state
    if op == 'int8':
        state['x'] = _activations(gen, (case['tokens'], case['inner'])).to(DTYPES[case['dtype']])
        state['weight'] = torch.randint(-127, 128, (case['outer'], case['inner']), generator=gen, device='cuda', dtype=torch.int8)
        state['channel_scale'] = (0.5 + torch.rand(case['outer'], generator=gen, device='cuda')) / (73.0 * math.sqrt(case['inner']))
        state['bias'] = 0.1 * torch.randn(case['outer'], generator=gen, device='cuda') if case['bias'] else None
        return state
    pairs = case['tokens'] * case['k']
    state['y'] = torch.randn(pairs, case['channels'], generator=gen, device='cuda').to(DTYPES[case['dtype']])
    gates = torch.rand(case['tokens'], case['k'], generator=gen, device='cuda') + 0.05
    slots = torch.randperm(pairs, generator=gen, device='cuda').view(case['tokens'], case['k']).to(torch.int32)
    pad = (torch.rand(case['tokens'], generator=gen, device='cuda') < case['padded'])[:, None]
    state['gates'] = torch.where(pad, 0.0, gates / gates.sum(1, keepdim=True))
    state['slots'] = torch.where(pad, -1, slots)
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _act(v, act):
    if act == 'relu':
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == 'silu':
        return v / (1.0 + torch.exp(-v))
    return v


def _plain_route(state):
    case, logits = state['case'], state['logits'].float()
    tokens, experts = logits.shape
    k = case['k']
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    best, index = torch.sort(logits, dim=1, descending=True, stable=True)               # equal values: lowest index first
    best, index = best[:, :k], index[:, :k]
    chosen = best > -math.inf
    weight = torch.where(chosen, torch.exp(best - best[:, :1]), 0.0)
    gates = torch.where(chosen, weight / weight.sum(1, keepdim=True), 0.0)
    flat = torch.where(chosen, index, experts).reshape(-1)
    by_expert, order = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(by_expert, torch.arange(experts + 1, device=flat.device))
    used = by_expert < experts
    slots = torch.empty_like(order)
    slots[order] = torch.where(used, torch.arange(tokens * k, device=flat.device), -1)
    return {'experts': torch.where(chosen, index, -1).to(torch.int32), 'gates': gates,
            'offsets': offsets.to(torch.int32), 'rows': torch.where(used, order // k, -1).to(torch.int32),
            'slots': slots.view(tokens, k).to(torch.int32)}


def _plain_grouped(state):
    case, offsets = state['case'], state['offsets'].long()
    x = state['x'] if state['rows'] is None else state['x'][state['rows'].long()]
    # sums of 8-bit products are whole numbers beyond the 24 bits of float32
    wide = torch.float64 if case['dtype'] == 'int8' else torch.float32
    total = x.shape[0]
    spread = offsets[:-1, None] + torch.arange(state['widest'], device=x.device)
    padded = x[spread.clamp(max=total - 1)].to(wide)                                    # [expert][row of its][inner]
    product = torch.bmm(padded, state['weight'].to(wide).transpose(1, 2))
    at = torch.arange(total, device=x.device)
    expert = torch.searchsorted(offsets[1:].contiguous(), at, right=True)
    v = product[expert, at - offsets[expert]]
    if state['row_scale'] is not None:
        scale = state['row_scale'] if state['rows'] is None else state['row_scale'][state['rows'].long()]
        v = v * scale[:, None] * state['channel_scale'][expert]
    if state['bias'] is not None:
        v = v + state['bias'][expert]
    if case['gated']:
        v = _act(v[:, :case['outer']], case['act']) * v[:, case['outer']:]
    else:
        v = _act(v, case['act'])
    return v.to(torch.bfloat16 if case['dtype'] == 'int8' else state['x'].dtype)


def _plain_int8(state):
    case, x = state['case'], state['x'].double()
    # in 64 bits: halves between two whole numbers decide the rounding, and the sums pass 24 bits
    largest = x.abs().amax(1, keepdim=True)
    q = torch.where(largest > 0, torch.round(x * 127.0 / largest), 0.0)
    scale = (largest / 127.0).float()
    v = torch.mm(q, state['weight'].double().t()).float() * scale * state['channel_scale']
    if state['bias'] is not None:
        v = v + state['bias']
    return _act(v, case['act']).to(state['x'].dtype)


def _plain_combine(state):
    slots = state['slots'].long()
    picked = state['y'][slots.clamp(min=0)].float()
    weighted = torch.where((slots >= 0)[:, :, None], picked * state['gates'][:, :, None], 0.0)
    return weighted.sum(1).to(state['y'].dtype)


# ---- the framework's operators ---------------------------------------------------------------------------------------

def _runtime():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'inter-operator-scheduler_b200')
    if not os.path.isdir(package):
        package = os.path.abspath('inter-operator-scheduler_b200')
    if package not in sys.path:
        sys.path.insert(0, package)
    from ios import ios_runtime
    return ios_runtime


def _own(state):
    rt, case = _runtime(), state['case']
    if case['op'] == 'route':
        routing = rt.route_experts(state['logits'], case['k'], renormalize=True)
        return {'experts': routing.experts, 'gates': routing.gates, 'offsets': routing.offsets, 'rows': routing.rows,
                'slots': routing.slots}
    if case['op'] == 'grouped':
        return rt.grouped_matmul(state['x'], state['weight'], state['offsets'], rows=state['rows'], bias=state['bias'],
                                 act=case['act'], gated=case['gated'], row_scale=state['row_scale'],
                                 channel_scale=state['channel_scale'],
                                 out_dtype=torch.bfloat16 if case['dtype'] == 'int8' else None)
    if case['op'] == 'int8':
        q, scale = rt.quantize_rows(state['x'])
        return rt.matmul_int8(q, state['weight'], scale, state['channel_scale'], bias=state['bias'], act=case['act'],
                              out_dtype=state['x'].dtype)
    return rt.combine_experts(state['y'], state['gates'], state['slots'])


def run(state):
    if own:
        return _own(state)
    return {'route': _plain_route, 'grouped': _plain_grouped, 'int8': _plain_int8,
            'combine': _plain_combine}[state['case']['op']](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    op = case['op']
    if op == 'route':
        size = 4 if case['dtype'] == 'fp32' else 2
        pairs = case['tokens'] * case['k']
        return {'bytes': case['tokens'] * case['experts'] * size + pairs * 16 + (case['experts'] + 1) * 4,
                'flops': case['tokens'] * case['experts'] * 2}
    if op == 'grouped':
        rows = case['tokens'] * case['k']
        size = {'bf16': 2, 'fp16': 2, 'fp32': 4, 'int8': 1}[case['dtype']]
        out = {'bf16': 2, 'fp16': 2, 'fp32': 4, 'int8': 2}[case['dtype']]
        busy = sum(1 for c in _loads(case) if c)
        channels = case['outer'] * (2 if case['gated'] else 1)
        total = busy * channels * case['inner'] * size + (case['tokens'] if case['gather'] else rows) * case['inner'] * size
        total += rows * case['outer'] * out + (case['experts'] + 1) * 4 + (rows * 4 if case['gather'] else 0)
        total += busy * channels * 4 if case['bias'] else 0
        total += rows * 4 + busy * channels * 4 if case['dtype'] == 'int8' else 0
        return {'bytes': total, 'flops': 2 * rows * channels * case['inner']}
    if op == 'int8':
        size = 4 if case['dtype'] == 'fp32' else 2
        total = case['tokens'] * (case['inner'] + case['outer']) * size + case['outer'] * (case['inner'] + 4)
        total += case['outer'] * 4 if case['bias'] else 0
        return {'bytes': total, 'flops': 2 * case['tokens'] * case['outer'] * case['inner']}
    size = 4 if case['dtype'] == 'fp32' else 2
    pairs = case['tokens'] * case['k']
    return {'bytes': pairs * case['channels'] * size + case['tokens'] * case['channels'] * size + pairs * 8,
            'flops': 2 * pairs * case['channels']}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def _exact_act(v, act):
    return {'identity': lambda t: t, 'relu': lambda t: t.clamp(min=0), 'silu': lambda t: t * torch.sigmoid(t)}[act](v)


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'route':
        # softmax over the k largest logits of a token; the plan itself is whole numbers
        logits = state['logits'].double()
        top = logits.topk(case['k'], dim=1).values
        gates = torch.softmax(top, dim=1).nan_to_num(0.0)
        return {'experts': None, 'gates': gates, 'offsets': None, 'rows': None, 'slots': None}
    if case['op'] == 'grouped':
        bounds = state['offsets'].tolist()
        out = torch.empty(case['tokens'] * case['k'], case['outer'], dtype=torch.float64, device='cuda')
        for e in range(case['experts']):
            b, t = bounds[e], bounds[e + 1]
            if b == t:
                continue
            mine = state['x'][b:t] if state['rows'] is None else state['x'].index_select(0, state['rows'][b:t].long())
            v = mine.double() @ state['weight'][e].double().mT
            if state['row_scale'] is not None:
                token_scale = state['row_scale'][b:t] if state['rows'] is None else state['row_scale'].index_select(0, state['rows'][b:t].long())
                v = v * torch.outer(token_scale.double(), state['channel_scale'][e].double())
            if state['bias'] is not None:
                v = v + state['bias'][e].double()
            if case['gated']:
                gate, up = v.chunk(2, dim=1)
                v = _exact_act(gate, case['act']) * up
            else:
                v = _exact_act(v, case['act'])
            out[b:t] = v
        return out
    if case['op'] == 'int8':
        x = state['x'].double()
        scale = x.abs().max(dim=1).values / 127.0
        # the multiple of the scale that is nearest, halves to even: 127 x over the row's largest magnitude
        q = torch.round((127.0 * x) / x.abs().max(dim=1).values[:, None]).nan_to_num(0.0)
        v = torch.einsum('tk,ok->to', q, state['weight'].double()) * torch.outer(scale, state['channel_scale'].double())
        if state['bias'] is not None:
            v = v + state['bias'].double()
        return _exact_act(v, case['act'])
    y, slots = state['y'].double(), state['slots'].long()
    out = torch.zeros(case['tokens'], case['channels'], dtype=torch.float64, device='cuda')
    for j in range(case['k']):
        live = slots[:, j] >= 0
        out[live] += y[slots[live, j]] * state['gates'][live, j, None].double()
    return out
