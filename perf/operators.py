"""The operators of a linear output layer over many classes, as they are timed:

  score     zs.linear_categorical_log_prob: log Categorical(y | X w^T + b) of given
            labels over a large vocabulary, whose logits are never kept
  train     the same with its gradients for X, w and b
  quantize  zs.quantize_rows and its values read back: 8-bit integers with one scale a row
  answer    zs.quantized_linear: X rounded to 8 bits a row, times 8-bit weights, scaled
            by token and channel

`run` computes them in plain torch, or calls the framework where `own` is true.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16}


def listed():
    """The cases; n: rows (tokens), d: features, v: classes (output channels)."""
    return [
        # 100 documents' topic vectors scored against the 12 419 words of the
        # topic model's corpus: the smallest call, latency
        dict(name='score_words', kind='score', dtype='float32', n=100, d=128, v=12419,
             bias=False, ignore=False),
        # one token of a sequence scored: the weights are read once
        dict(name='score_token', kind='score', dtype='bfloat16', n=1, d=4096, v=32768,
             bias=False, ignore=False),
        # a held-out set scored in one call
        dict(name='score_heldout', kind='score', dtype='bfloat16', n=5000, d=1024, v=50000,
             bias=True, ignore=True),
        # float32 training step at the width of an image's 784 pixels and the
        # corpus' vocabulary; odd sizes, a bias, some rows left out
        dict(name='train_ragged', kind='train', dtype='float32', n=1021, d=784, v=12419,
             bias=True, ignore=True),
        # an ordinary bfloat16 training step
        dict(name='train_batch', kind='train', dtype='bfloat16', n=4096, d=2048, v=32768,
             bias=False, ignore=True),
        # the largest: a long batch and a vocabulary of 2^17
        dict(name='train_large', kind='train', dtype='bfloat16', n=8192, d=4096, v=131072,
             bias=False, ignore=False),
        # the test images of a softmax regression, rounded to 8 bits
        dict(name='quantize_images', kind='quantize', dtype='float32', n=10000, d=784),
        # a whole output layer's weights, laid out once
        dict(name='quantize_weights', kind='quantize', dtype='bfloat16', n=131072, d=4096),
        # one token answered: the weights' bytes are the time
        dict(name='answer_token', kind='answer', dtype='bfloat16', n=1, d=4096, v=32768,
             bias=False),
        # a few rows, odd sizes, float32 in and out
        dict(name='answer_few', kind='answer', dtype='float32', n=13, d=1000, v=12419,
             bias=True),
        # a batch of requests that decode together
        dict(name='answer_batch', kind='answer', dtype='bfloat16', n=384, d=4096, v=16384,
             bias=False),
        # a long input in one call
        dict(name='answer_long', kind='answer', dtype='bfloat16', n=8192, d=8192, v=16384,
             bias=True),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ranges."""
    kind = rng.choice(['score', 'train', 'quantize', 'answer'])
    dtype = rng.choice(['float32', 'bfloat16'])
    case = dict(kind=kind, dtype=dtype)
    if kind == 'quantize':
        case.update(n=_between(rng, 1, 131072), d=_between(rng, 64, 4096))
        return case
    case.update(n=_between(rng, 1, 8192), d=_between(rng, 64, 4096), v=_between(rng, 500, 65536),
                bias=rng.random() < 0.5)
    if kind != 'answer':
        case.update(ignore=rng.random() < 0.5)
    if rng.random() < 0.5:      # half of the widths are a multiple of 64, as most layers' are
        case['d'] = max(64, case['d'] // 64 * 64)
    return case


def prepare(case, seed):
    """Inputs on the GPU, from the seed alone."""
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    dtype, n, d = DTYPES[case['dtype']], case['n'], case['d']

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device='cuda')

    state = dict(kind=case['kind'], dtype=dtype)
    if case['kind'] == 'quantize':
        # rows of different sizes, as activations and weights have them
        state['x'] = (normal(n, d) * torch.exp(0.5 * normal(n, 1))).to(dtype)
        return state
    v = case['v']
    w = normal(v, d) * (2.0 / math.sqrt(d))
    state['bias'] = 0.5 * normal(v) if case['bias'] else None
    if case['kind'] == 'answer':
        # the weights as a program keeps them: 8-bit rows at a pitch of whole
        # 128 bytes, one scale an output channel
        scale = w.abs().amax(1) / 127.0
        pitch = (d + 127) // 128 * 128
        values = torch.zeros(v, pitch, dtype=torch.int8, device='cuda')
        values[:, :d] = torch.round(w / scale[:, None]).to(torch.int8)
        state.update(x=normal(n, d).to(dtype), values=values[:, :d], scale=scale)
        return state
    labels = torch.randint(v, (n,), generator=gen, device='cuda')
    # a model that has learnt something: a row's features point at its label
    # by a factor that differs from row to row
    pull = 1.5 * torch.rand(n, 1, generator=gen, device='cuda')
    state['x'] = (normal(n, d) + pull * w[labels]).to(dtype)
    state['w'] = w.to(dtype)
    if case['ignore']:          # padding and prompts: left out of the sum
        out = torch.rand(n, generator=gen, device='cuda') < 0.15
        labels = torch.where(out, torch.full_like(labels, IGNORE), labels)
    state['labels'], state['ignore'] = labels, case['ignore']
    if case['kind'] == 'train':
        # the gradient of a weighted mean over the rows
        state['grad'] = (0.5 + torch.rand(n, generator=gen, device='cuda')) / n
    return state


def run(state):
    """One pass."""
    return _own(state) if own else _plain(state)


def _own(state):
    import zhusuan_amd as zs
    kind, x = state['kind'], state['x']
    if kind == 'quantize':
        rows = zs.quantize_rows(x)
        return [rows.dequantize(), rows.scale]
    if kind == 'answer':
        w = zs.QuantizedRows(state['values'], state['scale'])
        return zs.quantized_linear(w, x, bias=state['bias'])
    ignore = IGNORE if state['ignore'] else None
    if kind == 'score':
        return zs.linear_categorical_log_prob(state['w'], x, state['labels'], bias=state['bias'],
                                              ignore_label=ignore)
    leaves = [t.detach().requires_grad_() for t in (x, state['w'], state['bias']) if t is not None]
    log_prob = zs.linear_categorical_log_prob(leaves[1], leaves[0], state['labels'],
                                              bias=leaves[2] if len(leaves) > 2 else None,
                                              ignore_label=ignore)
    return [log_prob.detach()] + list(torch.autograd.grad(log_prob, leaves, state['grad']))


def _rounded(x):
    """(whole numbers in [-127, 127] as float32, scale) of the rows of x."""
    x = x.float()
    most = x.abs().amax(1, keepdim=True)
    # (a tensor: a division by a Python number is a product with its reciprocal)
    scale = most / torch.full_like(most, 127.0)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(x / scale).clamp(-127, 127), scale


def _plain(state):
    kind, dtype, x = state['kind'], state['dtype'], state['x']
    if kind == 'quantize':
        values, scale = _rounded(x)
        return [values * scale, scale[:, 0]]
    bias = state['bias']
    if kind == 'answer':
        values, scale = _rounded(x)
        out = values @ state['values'].float().t() * (scale * state['scale'])
        return (out if bias is None else out + bias).to(dtype)
    labels, w = state['labels'], state['w'].float()
    x = x.float()
    logits = x @ w.t()
    if bias is not None:
        logits = logits + bias
    kept = labels != IGNORE
    index = torch.where(kept, labels, torch.zeros_like(labels))[:, None]
    most = logits.amax(1, keepdim=True)
    log_sum = most + torch.log(torch.exp(logits - most).sum(1, keepdim=True))
    log_prob = torch.where(kept, (logits.gather(1, index) - log_sum)[:, 0],
                           torch.zeros_like(log_sum[:, 0]))
    if kind == 'score':
        return log_prob
    g = torch.where(kept, state['grad'], torch.zeros_like(state['grad']))[:, None]
    r = torch.exp(logits - log_sum) * -g
    r.scatter_add_(1, index, g)
    out = [log_prob, (r @ w).to(dtype), (r.t() @ x).to(dtype)]
    return out if bias is None else out + [r.sum(0)]


def work(case):
    """Each input read and each output written once; the products that no form can do without."""
    n, d, kind = case['n'], case['d'], case['kind']
    size = 4 if case['dtype'] == 'float32' else 2
    if kind == 'quantize':
        return dict(bytes=n * d * (size + 4) + 4 * n, flops=3 * n * d)
    v = case['v']
    if kind == 'answer':
        return dict(bytes=n * d * size + v * d + 4 * v * (1 + case['bias']) + n * v * size,
                    flops=2 * n * v * d)
    read = (n + v) * d * size + 8 * n + 4 * v * case['bias']
    if kind == 'score':
        return dict(bytes=read + 4 * n, flops=2 * n * v * d)
    return dict(bytes=read + 8 * n + (n + v) * d * size + 4 * v * case['bias'],
                flops=6 * n * v * d)


def exact(case, seed):
    """The outputs in 64 bits. A scale is by definition a float32 number, and so is the quotient
    that is rounded to a whole number (to the even one of two that are as near)."""
    state = prepare(case, seed)
    x = state['x'].double()
    if case['kind'] in ('quantize', 'answer'):
        scale = (x.abs().max(dim=1).values / 127).float().double()
        scale[scale == 0] = 1
        x.div_(scale[:, None])
        values = x.float().round_().double()
        if case['kind'] == 'quantize':
            return [values.mul_(scale[:, None]), scale]
        out = torch.matmul(values, state['values'].double().t())
        out.mul_(scale[:, None]).mul_(state['scale'].double())
        return out if state['bias'] is None else out.add_(state['bias'].double())
    w, labels = state['w'].double(), state['labels']
    logits = torch.matmul(x, w.t())
    if state['bias'] is not None:
        logits.add_(state['bias'].double())
    rows = torch.nonzero(labels >= 0)[:, 0]
    log_p = logits.sub_(torch.logsumexp(logits, dim=1)[:, None])
    log_prob = torch.zeros(case['n'], dtype=torch.float64, device='cuda')
    log_prob[rows] = log_p[rows, labels[rows]]
    if case['kind'] == 'score':
        return log_prob
    r = log_p.exp_().neg_()
    r[rows, labels[rows]] += 1
    grad = torch.zeros_like(log_prob)
    grad[rows] = state['grad'].double()[rows]
    r.mul_(grad[:, None])
    out = [log_prob, torch.matmul(r, w), torch.matmul(r.t(), x)]
    return out if state['bias'] is None else out + [r.sum(dim=0)]
