"""The operators that shared codes and tokens are learned with, as cases to be timed and compared: the softmax cross entropy of
rows against every row of a table, without the logits in memory (`efgs.linear_cross_entropy`), dropout by a counter-based
generator, whose mask is never stored (`efgs.dropout`), and the loss that balances how often codes or experts are chosen, with
their counts (`efgs.balance_loss`).

`run` computes them from elementary torch operations where `own` is false, and through the framework's entry points where it
is true. `listed` gives the standing cases, `draw` more of the same ranges, `exact` the same results in 64 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _efgs():
    package = str(Path(__file__).resolve().parent.parent / 'efficient-gaussian-appearance_amd')
    if package not in sys.path:
        sys.path.insert(0, package)
    import efgs
    return efgs


def entropy(n, rows, columns, dtype='bf16', train=True, reduction='mean', scale=1.0, left_out=0.0):
    return dict(kind='entropy', n=n, rows=rows, columns=columns, dtype=dtype, train=train, reduction=reduction, scale=scale, left_out=left_out)


def drop(n, columns, p, dtype='bf16', train=True, residual=False):
    return dict(kind='dropout', n=n, columns=columns, p=p, dtype=dtype, train=train, residual=residual)


def balance(n, experts, chosen, dtype='f32', train=True, left_out=0.0):
    return dict(kind='balance', n=n, experts=experts, chosen=chosen, dtype=dtype, train=train, left_out=left_out)


def listed():
    return [
        # answering: how likely one token was, against the whole table; the table's bytes are what counts
        dict(entropy(1, 49_999, 4096, train=False, reduction='none'), name='entropy_score_1_token'),
        # scoring a short answer: odd sizes, each row's own loss
        dict(entropy(37, 30_011, 1000, 'f16', train=False, reduction='none', left_out=0.1), name='entropy_score_37_tokens'),
        # training of a small head, padding among the tokens
        dict(entropy(2_047, 49_999, 1024, left_out=0.05), name='entropy_train_2k_tokens'),
        # training of a large head: matrix products are all that counts
        dict(entropy(8_192, 128_000, 4096), name='entropy_train_8k_tokens'),
        # training with a weight for each row, sizes that no tile divides
        dict(entropy(1_001, 10_007, 333, 'f16', reduction='none', scale=0.7), name='entropy_train_odd_f16'),
        # every primitive's features against a codebook, at a temperature
        dict(entropy(1_000_000, 4096, 8, 'f32', scale=8.0, left_out=0.02), name='entropy_train_1m_codes'),
        # training: dropout of the code features of a million primitives
        dict(drop(1_000_000, 8, 0.1, 'f32'), name='dropout_train_1m_codes'),
        # training: dropout of a block's output, added to what went past the block
        dict(drop(16_383, 4096, 0.1, residual=True), name='dropout_train_16k_tokens'),
        # a few rows: launches and host time count
        dict(drop(5, 1000, 0.5, 'f16'), name='dropout_train_5_rows'),
        # training: a million primitives over a small codebook, one code each
        dict(balance(1_000_000, 64, 1, left_out=0.02), name='balance_train_1m_codes'),
        # training: a step's tokens over many experts, eight for each
        dict(balance(16_383, 250, 8, 'bf16', left_out=0.05), name='balance_train_16k_tokens'),
        # a few tokens: launches and host time count
        dict(balance(9, 60, 4), name='balance_train_9_tokens'),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(('tokens', 'tokens', 'score', 'codes', 'dropout', 'dropout', 'balance', 'balance'))
    if kind == 'score':
        dtype, columns = rng.choice((('bf16', _log_uniform(rng, 64, 4096)), ('f16', _log_uniform(rng, 64, 4096)), ('f32', _log_uniform(rng, 8, 1024))))
        return entropy(_log_uniform(rng, 1, 300), _log_uniform(rng, 500, 130_000), columns, dtype, False, rng.choice(('none', 'sum')),
                       round(rng.uniform(0.5, 1.5), 3), rng.choice((0.0, 0.1)))
    if kind == 'tokens':
        columns, rows = _log_uniform(rng, 130, 4096), _log_uniform(rng, 300, 100_000)
        n = _log_uniform(rng, 20, min(8_000, int(1.2e12 / (columns * rows)) + 21))
        return entropy(n, rows, columns, rng.choice(('bf16', 'bf16', 'f16')), True, rng.choice(('mean', 'sum', 'none')),
                       round(rng.uniform(0.5, 1.5), 3), rng.choice((0.0, 0.05, 0.5)))
    if kind == 'codes':
        columns, rows = rng.choice((3, 8, 16, 45, 48, 64, 200)), _log_uniform(rng, 16, 20_000)
        n = _log_uniform(rng, 1_000, min(1_000_000, int(2.5e10 / (columns * rows)) + 1_001))
        return entropy(n, rows, columns, rng.choice(('f32', 'f32', 'bf16')), True, rng.choice(('mean', 'none')), round(rng.uniform(1.0, 10.0), 3),
                       rng.choice((0.0, 0.02)))
    if kind == 'dropout':
        dtype = rng.choice(tuple(DTYPES))
        columns = rng.choice((3, 8, 45, 64, 1000, 1024, 4096))
        return drop(_log_uniform(rng, 1, 60_000_000 // columns), columns, rng.choice((0.05, 0.1, 0.25, 0.5)), dtype, rng.random() < 0.7, rng.random() < 0.4)
    experts = _log_uniform(rng, 2, 4096)
    return balance(_log_uniform(rng, 1, min(1_000_000, 60_000_000 // experts)), experts, rng.randint(1, min(8, experts)), rng.choice(tuple(DTYPES)),
                   rng.random() < 0.7, rng.choice((0.0, 0.05)))


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator('cuda').manual_seed(int(seed) & 0x7fffffff)


def _entropy_inputs(case, seed):
    """Rows that point towards their target's table row, from not at all to nearly sure; each row's upstream gradient."""
    g, n, rows, columns, dtype = _generator(seed), case['n'], case['rows'], case['columns'], DTYPES[case['dtype']]
    # (logits: deviation 2 beside the target's)
    table = (torch.randn((rows, columns), generator=g, device='cuda') * (2.0 / (case['scale'] * math.sqrt(columns)))).to(dtype)
    targets = (rows * torch.rand(n, generator=g, device='cuda', dtype=torch.float64) ** 2).long().clamp(max=rows - 1)
    pull = torch.rand(n, generator=g, device='cuda') * (16.0 * case['scale'] / 4.0)
    features = (torch.randn((n, columns), generator=g, device='cuda') + pull[:, None] * table[targets].float()).to(dtype)
    weights = torch.rand(n, generator=g, device='cuda') + 0.1
    if case['left_out']:
        targets[torch.rand(n, generator=g, device='cuda') < case['left_out']] = -1
    return features, table, targets, weights


def _dropout_inputs(case, seed):
    g, dtype, shape = _generator(seed), DTYPES[case['dtype']], (case['n'], case['columns'])
    x, upstream, residual = (torch.randn(shape, generator=g, device='cuda').to(dtype) for _ in range(3))
    key = int(torch.randint(0, 2 ** 62, (), generator=torch.Generator().manual_seed(int(seed) & 0x7fffffff)))
    return x, residual if case['residual'] else None, upstream, key


def _balance_inputs(case, seed):
    """Logits that favour some of the experts, and the experts of the largest ones."""
    g, n, experts = _generator(seed), case['n'], case['experts']
    logits = torch.randn((n, experts), generator=g, device='cuda') * 1.5 + torch.randn(experts, generator=g, device='cuda')
    logits = logits.to(DTYPES[case['dtype']])
    indices = logits.float().topk(case['chosen'], dim=1).indices
    if case['left_out']:
        indices[torch.rand(n, generator=g, device='cuda') < case['left_out']] = -1
    return logits, indices, 0.25 + torch.rand((), generator=g, device='cuda')


def prepare(case, seed):
    if own:
        _efgs()
    if case['kind'] == 'entropy':
        features, table, targets, weights = _entropy_inputs(case, seed)
        return dict(case=case, features=features.requires_grad_(case['train']), table=table.requires_grad_(case['train']), targets=targets,
                    upstream=weights if case['reduction'] == 'none' else weights[0].clone())
    if case['kind'] == 'dropout':
        x, residual, upstream, key = _dropout_inputs(case, seed)
        return dict(case=case, x=x.requires_grad_(case['train']), residual=None if residual is None else residual.requires_grad_(case['train']),
                    upstream=upstream, seed=key, offset=3)
    logits, indices, upstream = _balance_inputs(case, seed)
    return dict(case=case, logits=logits.requires_grad_(case['train']), indices=indices, upstream=upstream)


# ---- the operators in plain form -------------------------------------------------------------------------------------
# Cross entropy: z = scale x . w, loss = log sum exp z - z[target]; a target outside the table leaves its row out; the mean is
# over the rows that count.

def _plain_entropy(state):
    case = state['case']
    x, w, targets, scale = state['features'].detach().float(), state['table'].detach().float(), state['targets'], case['scale']
    n, rows = case['n'], case['rows']
    counted = (targets >= 0) & (targets < rows)
    mean = 1.0 / counted.sum().clamp(min=1).float() if case['reduction'] == 'mean' else torch.ones((), device='cuda')
    upstream = state['upstream'] * mean * counted
    losses = torch.empty(n, device='cuda')
    grad_x, grad_w = (torch.zeros_like(x), torch.zeros_like(w)) if case['train'] else (None, None)
    step = max(1, (1 << 28) // rows)
    for a in range(0, n, step):
        part, hit = slice(a, min(n, a + step)), counted[a:a + step]
        target = targets[part].clamp(0, rows - 1)[:, None]
        z = (x[part] @ w.T) * scale
        top = z.amax(1, keepdim=True)
        own_logit = z.gather(1, target)
        z = (z - top).exp_()
        total = z.sum(1, keepdim=True)
        losses[part] = ((total.log() + top - own_logit)[:, 0] * hit)
        if case['train']:
            z = z / total
            z.scatter_add_(1, target, torch.full_like(total, -1.0))
            z *= upstream[part, None]
            grad_x[part] = (z @ w) * scale
            grad_w += z.T @ (x[part] * scale)
    loss = losses if case['reduction'] == 'none' else losses.sum() * mean
    if not case['train']:
        return dict(loss=loss)
    return dict(loss=loss, grad_features=grad_x.to(state['features'].dtype), grad_table=grad_w.to(state['table'].dtype))


# Dropout: Philox4x32-10 of the counter (index / 8, offset) and the key seed gives 16 bits for each of eight elements; one below
# round(65536 p) drops its element, the others are divided by what is kept of 65536.

PHILOX = (0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85)


def _bits(n, seed, offset):
    """16 random bits for each of n elements."""
    at = torch.arange((n + 7) // 8, device='cuda')
    c0, c1 = at & 0xffffffff, at >> 32
    c2, c3 = torch.full_like(at, offset & 0xffffffff), torch.full_like(at, offset >> 32)
    k0, k1 = seed & 0xffffffff, seed >> 32
    for _ in range(10):
        a, b = c0 * PHILOX[0], c2 * PHILOX[1]   # (whole 64-bit products)
        c0, c1, c2, c3 = ((b >> 32) & 0xffffffff) ^ c1 ^ k0, b & 0xffffffff, ((a >> 32) & 0xffffffff) ^ c3 ^ k1, a & 0xffffffff
        k0, k1 = (k0 + PHILOX[2]) & 0xffffffff, (k1 + PHILOX[3]) & 0xffffffff
    words = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((words & 0xffff, words >> 16), 2).view(-1)[:n]


def _plain_dropout(state):
    case, x, upstream = state['case'], state['x'].detach(), state['upstream']
    threshold = round(case['p'] * 65536)
    kept = (_bits(x.numel(), state['seed'], state['offset']) >= threshold).view(x.shape)
    scale = 65536.0 / (65536 - threshold)
    zero = torch.zeros((), device='cuda')
    out = torch.where(kept, x.float() * scale, zero)
    out = (out if state['residual'] is None else out + state['residual'].detach().float()).to(x.dtype)
    if not case['train']:
        return dict(out=out)
    grad = torch.where(kept, upstream.float() * scale, zero).to(x.dtype)
    return dict(out=out, grad_x=grad) if state['residual'] is None else dict(out=out, grad_x=grad, grad_residual=upstream)


# Balance: over the rows with a chosen expert, E times the sum over the experts of (share of the choices) x (mean probability).

def _plain_balance(state):
    case, logits, indices, experts = state['case'], state['logits'].detach().float(), state['indices'], state['case']['experts']
    chosen = (indices >= 0) & (indices < experts)
    row = chosen.any(1)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device='cuda').index_add_(
        0, torch.where(chosen, indices, experts).view(-1), torch.ones(indices.numel(), dtype=torch.int64, device='cuda'))[:experts]
    share = counts.float() / counts.sum().clamp(min=1).float()
    p = (logits - logits.amax(1, keepdim=True)).exp()
    p = p / p.sum(1, keepdim=True)
    p = p * row[:, None]
    rows = row.sum().clamp(min=1)
    mean = (p.sum(0, dtype=torch.float64) / rows).float()
    loss = (share * mean).sum() * experts
    if not case['train']:
        return dict(loss=loss, counts=counts)
    grad = p * (share - (p * share).sum(1, keepdim=True)) * (state['upstream'] * experts / rows.float())
    return dict(loss=loss, counts=counts, grad=grad.to(state['logits'].dtype))


def run(state):
    case = state['case']
    if not own:
        with torch.no_grad():
            return {'entropy': _plain_entropy, 'dropout': _plain_dropout, 'balance': _plain_balance}[case['kind']](state)
    efgs = _efgs()
    if case['kind'] == 'entropy':
        loss = efgs.linear_cross_entropy(state['features'], state['table'], state['targets'], scale=case['scale'], reduction=case['reduction'])
        if not case['train']:
            return dict(loss=loss)
        grads = torch.autograd.grad(loss, (state['features'], state['table']), state['upstream'])
        return dict(loss=loss.detach(), grad_features=grads[0], grad_table=grads[1])
    if case['kind'] == 'dropout':
        out = efgs.dropout(state['x'], case['p'], seed=state['seed'], offset=state['offset'], residual=state['residual'])
        if not case['train']:
            return dict(out=out)
        if state['residual'] is None:
            return dict(out=out.detach(), grad_x=torch.autograd.grad(out, state['x'], state['upstream'])[0])
        grads = torch.autograd.grad(out, (state['x'], state['residual']), state['upstream'])
        return dict(out=out.detach(), grad_x=grads[0], grad_residual=grads[1])
    loss, counts = efgs.balance_loss(state['logits'], state['indices'])
    if not case['train']:
        return dict(loss=loss, counts=counts)
    return dict(loss=loss.detach(), counts=counts, grad=torch.autograd.grad(loss, state['logits'], state['upstream'])[0])


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    size, n = DTYPES[case['dtype']].itemsize, case['n']
    if case['kind'] == 'entropy':
        rows, columns = case['rows'], case['columns']
        inputs = size * columns * (n + rows) + 8 * n
        # products: the logits; with gradients those of the rows and of the table too
        if case['train']:
            return dict(bytes=inputs + size * columns * (n + rows), flops=6 * n * rows * columns)
        return dict(bytes=inputs + 4 * n, flops=2 * n * rows * columns)
    if case['kind'] == 'dropout':
        elements = n * case['columns']
        arrays = (4 if case['train'] else 2) + (1 if case['residual'] else 0)
        return dict(bytes=arrays * size * elements, flops=2 * elements)
    elements = n * case['experts']
    return dict(bytes=8 * n * case['chosen'] + size * elements * (2 if case['train'] else 1) + 8 * case['experts'], flops=8 * elements)


# ---- the same in 64 bits -------------------------------------------------------------------------------------------------

def _exact_entropy(case, seed):
    features, table, targets, weights = _entropy_inputs(case, seed)
    x, w, n = features.double() * case['scale'], table.double(), case['n']
    inside = (targets >= 0) & (targets < case['rows'])
    share = 1.0 / max(1, int(inside.sum())) if case['reduction'] == 'mean' else 1.0
    losses = torch.zeros(n, dtype=torch.float64, device='cuda')
    grad_x, grad_w = torch.zeros_like(x), torch.zeros_like(w)
    for rows in torch.arange(n, device='cuda')[inside].split(max(1, (1 << 27) // case['rows'])):
        logits, target = torch.mm(x[rows], w.t()), targets[rows]
        total = torch.logsumexp(logits, dim=1)
        at = torch.arange(len(rows), device='cuda')
        losses[rows] = total - logits[at, target]
        if case['train']:
            p = torch.exp(logits - total.unsqueeze(1))
            p[at, target] -= 1.0
            p *= (weights[rows].double() if case['reduction'] == 'none' else weights[0].double()).view(-1, 1) * share
            grad_x[rows] = torch.mm(p, w) * case['scale']
            grad_w += torch.mm(p.t(), x[rows])
    out = dict(loss=losses if case['reduction'] == 'none' else losses.sum() * share)
    return dict(out, grad_features=grad_x, grad_table=grad_w) if case['train'] else out


def _exact_dropout(case, seed):
    x, residual, upstream, key = _dropout_inputs(case, seed)
    # (the generator's words from 16-bit halves: a = m x high and low word without a 64-bit product)
    def product(x, m):
        low, high = (x & 0xffff) * m, (x >> 16) * m
        low = low + ((high & 0xffff) << 16)
        return (high >> 16) + (low >> 32), low & 0xffffffff
    index = torch.arange(x.numel(), device='cuda')
    group, half = torch.div(index, 8, rounding_mode='floor'), index % 8
    group = group[::8]
    words, offset = [group % 2 ** 32, group // 2 ** 32, torch.full_like(group, 3), torch.zeros_like(group)], 0
    for _ in range(10):
        (h0, l0), (h1, l1) = product(words[0], 0xD2511F53), product(words[2], 0xCD9E8D57)
        words = [h1 ^ words[1] ^ ((key + offset * 0x9E3779B9) % 2 ** 32), l1, h0 ^ words[3] ^ (((key >> 32) + offset * 0xBB67AE85) % 2 ** 32), l0]
        offset += 1
    dropped = torch.empty(x.numel(), dtype=torch.bool, device='cuda')
    for k in range(8):
        at = half == k
        dropped[at] = ((words[k // 2] >> (16 * (k % 2))) % 65536)[:int(at.sum())] < round(case['p'] * 65536)
    factor = 1.0 / (1.0 - round(case['p'] * 65536) / 65536)
    out = (x.double() * factor).masked_fill(dropped.view(x.shape), 0.0)
    if residual is not None:
        out = out + residual.double()
    if not case['train']:
        return dict(out=out)
    grad = (upstream.double() * factor).masked_fill(dropped.view(x.shape), 0.0)
    return dict(out=out, grad_x=grad) if residual is None else dict(out=out, grad_x=grad, grad_residual=upstream.double())


def _exact_balance(case, seed):
    logits, indices, upstream = _balance_inputs(case, seed)
    experts = case['experts']
    valid = indices[(indices >= 0) & (indices < experts)]
    counts = torch.bincount(valid, minlength=experts)
    rows = ((indices >= 0) & (indices < experts)).sum(1) > 0
    share = counts.double() / max(1, valid.numel())
    p = torch.softmax(logits.double(), dim=1) * rows.double().unsqueeze(1)
    number = max(1, int(rows.sum()))
    loss = experts * (p.mean(0) * (case['n'] / number) * share).sum()
    if not case['train']:
        return dict(loss=loss, counts=counts)
    weighted = torch.mv(p, share).unsqueeze(1)
    return dict(loss=loss, counts=counts, grad=upstream.double() * (experts / number) * p * (share.unsqueeze(0) - weighted))


def exact(case, seed):
    return {'entropy': _exact_entropy, 'dropout': _exact_dropout, 'balance': _exact_balance}[case['kind']](case, seed)
