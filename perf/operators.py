"""Cases of the 8-bit encoder operators: the matrix product in 8-bit integers with a scale
per token and per channel, and the group norm with an activation (channels last).

``run`` computes a case in plain torch operations, or, with ``own`` set, through the public
entry points (``Runtime.linear_i8``, ``Runtime.group_norm``, ``Runtime.group_norm_quantize``).

Definitions. A token row x is quantised with s = max|x| / 127 rounded to fp32 and
q = x / s rounded to the nearest integer, ties to even (values next to a border are decided by the exact
quotient, hence 64 bits in the plain form). The product is the exact integer sum of q times the
8-bit weights, scaled by s and by the channel's scale; bias, activation or residual follow and the
result is rounded once to the output's type. The group norm takes mean and (biased) variance over
the frames of one window and the channels of one group.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
EPS = 1e-5
_runtime = None


# ---------------------------------------------------------------------------- cases
def _linear(name, m, k, n, epi='none', x='f32', y='f32', norm=False, bias=True):
    return {'name': name, 'op': 'linear', 'm': m, 'k': k, 'n': n, 'epi': epi, 'x': x, 'y': y, 'norm': norm,
            'bias': bias}


def _norm(name, windows, t, channels, groups, act='silu', x='f32', ragged=False):
    return {'name': name, 'op': 'group_norm', 'windows': windows, 't': t, 'channels': channels, 'groups': groups,
            'act': act, 'x': x, 'ragged': ragged}


def listed():
    return [
        # one frame of one stream through FFN linear1: latency of a single call
        _linear('linear_1x1024x4096_silu', 1, 1024, 4096, 'silu'),
        # the joint's output layer (8193 tokens + 5 durations) for eight streams
        _linear('linear_8x640x8198_bf16', 8, 640, 8198, 'none', 'bf16', 'f32'),
        # FFN linear2 for a short chunk of frames: long K, few rows, residual
        _linear('linear_45x4096x1024_resid', 45, 4096, 1024, 'residual', 'bf16', 'bf16'),
        # one 30 s window through LayerNorm and pointwise_conv1 with its GLU
        _linear('ln_linear_375x1024x2048_glu', 375, 1024, 2048, 'glu', 'f32', 'f32', True, False),
        # a ragged number of frames, the joint's width: no dimension a multiple of a tile
        _linear('linear_1499x640x8198_f16', 1499, 640, 8198, 'relu', 'f16', 'f16'),
        # eight windows through FFN linear2 with the half residual, fp32 stream
        _linear('linear_3000x4096x1024_resid', 3000, 4096, 1024, 'residual', 'f32', 'f32', False, False),
        # sixty-four windows through LayerNorm and FFN linear1 + SiLU
        _linear('ln_linear_24000x1024x4096', 24000, 1024, 4096, 'silu', 'f32', 'bf16', True),
        # a streaming chunk of seven frames: latency of a single group norm
        _norm('group_norm_1x7x1024', 1, 7, 1024, 32),
        # the conv module's norm over eight windows of 30 s
        _norm('group_norm_8x375x1024', 8, 375, 1024, 32),
        # windows of unequal lengths, a channel count with odd groups, a half type
        _norm('group_norm_ragged_1000', 13, 613, 1000, 8, 'none', 'f16', True),
        # sixty-four windows, one group per window (layer-wise statistics)
        _norm('group_norm_64x375x1024_g1', 64, 375, 1024, 1, 'silu', 'bf16'),
        # the conv module's tail over eight windows: group norm + SiLU quantised, pointwise_conv2 + residual
        {'name': 'norm_linear_8x375x1024', 'op': 'norm_linear', 'windows': 8, 't': 375, 'channels': 1024,
         'groups': 32, 'n': 1024, 'x': 'f32', 'ragged': False},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['linear', 'linear', 'linear', 'group_norm', 'group_norm', 'norm_linear'])
    types = ['f32', 'f16', 'bf16']
    if op == 'linear':
        epi = rng.choice(['none', 'relu', 'silu', 'glu', 'residual'])
        k = 16 * rng.randint(1, 256)
        n = rng.choice([rng.randint(1, 8198), 256 * rng.randint(1, 16)])
        n += n % 2 if epi == 'glu' else 0
        m = _log_uniform(rng, 1, 24000)
        while m * k * n > 24000 * 1024 * 4096:
            m = (m + 1) // 2
        return {'op': op, 'm': m, 'k': k, 'n': n, 'epi': epi, 'x': rng.choice(types), 'y': rng.choice(types),
                'norm': rng.random() < 0.4, 'bias': rng.random() < 0.6}
    groups = rng.choice([1, 2, 4, 8, 16, 32])
    width = rng.randint(1, 2048 // groups)
    if op == 'norm_linear':
        groups, width = rng.choice([1, 8, 16, 32]), 16 * rng.randint(1, 4)
    windows = _log_uniform(rng, 1, 64)
    t = _log_uniform(rng, 1, 5000)
    while windows * t * groups * width > 24000 * 1024:
        t = (t + 1) // 2
    c = {'op': op, 'windows': windows, 't': t, 'channels': groups * width, 'groups': groups,
         'x': rng.choice(types), 'ragged': rng.random() < 0.5}
    if op == 'group_norm':
        c['act'] = rng.choice(['none', 'relu', 'silu'])
    else:
        c['n'] = rng.randint(1, 2048)
    return c


# ---------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device='cuda')


def _weight(g, n, k):
    """8-bit weight rows with a scale per channel, as quantising a trained matrix per channel gives them."""
    q = (_normal(g, n, k) * 32).round_().clamp_(-127, 127).to(torch.int8)
    scale = torch.exp(0.3 * _normal(g, n)) * (0.6 / 32 / math.sqrt(k))
    return q, scale


def _tokens(g, rows, width, dtype):
    """Activations: token magnitudes spread over a factor of a few, a few loud channels, a common offset."""
    x = _normal(g, rows, width) * torch.exp(0.5 * _normal(g, rows, 1)) * torch.exp(0.5 * _normal(g, 1, width))
    return (x + 0.25 * _normal(g, 1, width)).to(dtype)


def _offsets(case, g):
    """Window boundaries (int32, on the device): equal ones, or lengths from a frame up, summing to windows * t."""
    windows, t = case['windows'], case['t']
    if not case['ragged']:
        return None
    cuts = torch.sort(torch.randint(0, windows * t + 1, (windows - 1,), generator=g, device='cuda'))[0]
    ends = torch.tensor([0, windows * t], device='cuda')
    return torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case['op'] == 'linear':
        m, k, n = case['m'], case['k'], case['n']
        s['x_t'] = _tokens(g, m, k, TYPES[case['x']])
        s['wq'], s['ws'] = _weight(g, n, k)
        s['b'] = 0.1 * _normal(g, n) if case['bias'] else None
        s['res'] = _normal(g, m, n).to(TYPES[case['y']]) if case['epi'] == 'residual' else None
        s['gamma'], s['beta'] = 1 + 0.1 * _normal(g, k), 0.1 * _normal(g, k)
    else:
        rows, c = case['windows'] * case['t'], case['channels']
        s['x_t'] = _tokens(g, rows, c, TYPES[case['x']])
        s['gamma'], s['beta'] = 1 + 0.1 * _normal(g, c), 0.1 * _normal(g, c)
        s['offsets'] = _offsets(case, g)
        if case['op'] == 'norm_linear':
            s['wq'], s['ws'] = _weight(g, case['n'], c)
            s['res'] = _normal(g, rows, case['n'])
    return s


# ---------------------------------------------------------------------------- plain form
def _quantized(h):
    """Row scales (fp32) and integers (held in 64 bits, where quotients next to a border stay on their side)."""
    h = h.double()
    scale = (h.abs().amax(1, keepdim=True) / 127).float()
    q = torch.where(scale > 0, torch.round(h / scale.double()), torch.zeros((), dtype=h.dtype, device=h.device))
    return q, scale


def _layer_norm(x, gamma, beta):
    x = x.double()
    d = x - x.mean(1, keepdim=True)
    return d * torch.rsqrt((d * d).mean(1, keepdim=True) + EPS) * gamma + beta


def _act(z, name):
    if name == 'relu':
        return torch.clamp(z, min=0)
    if name == 'silu':
        return z / (1 + torch.exp(-z))
    return z


def _product(h, wq, ws, b, epi, res, alpha, dtype):
    q, scale = _quantized(h)
    acc = q @ wq.double().t()  # whole numbers up to 127 * 127 * k: exact in 64 bits, not in 32
    z = (acc * scale).float() * ws
    if b is not None:
        z = z + b
    if epi == 'glu':
        half = z.shape[1] // 2
        z = z[:, :half] / (1 + torch.exp(-z[:, half:]))
    elif epi == 'residual':
        z = res.float() + alpha * z
    else:
        z = _act(z, epi)
    return z.to(dtype)


def _segments(s):
    """Window number of every row and the number of rows of every window."""
    rows = s['windows'] * s['t']
    at = torch.arange(rows, device='cuda')
    if s['offsets'] is None:
        return at // s['t'], torch.full((s['windows'],), s['t'], device='cuda')
    ends = s['offsets'][1:].long()
    return torch.searchsorted(ends, at, right=True), ends - s['offsets'][:-1].long()


def _group_norm(s, act):
    rows, c = s['x_t'].shape
    groups, windows = s['groups'], s['windows']
    window, length = _segments(s)
    x = s['x_t'].double().view(rows, groups, c // groups)  # sums over thousands of frames: in 64 bits
    count = (length.clamp(min=1) * (c // groups)).double()[:, None]
    zero = torch.zeros(windows, groups, dtype=torch.float64, device='cuda')
    mean = zero.index_add(0, window, x.sum(2)) / count
    d = x - mean[window][:, :, None]
    var = zero.index_add(0, window, (d * d).sum(2)) / count
    h = (d * torch.rsqrt(var + EPS)[window][:, :, None]).view(rows, c) * s['gamma'] + s['beta']
    return _act(h, act)


def _plain(s):
    if s['op'] == 'linear':
        h = _layer_norm(s['x_t'], s['gamma'], s['beta']) if s['norm'] else s['x_t']
        return _product(h, s['wq'], s['ws'], s['b'], s['epi'], s['res'], 0.5, TYPES[s['y']])
    if s['op'] == 'group_norm':
        return _group_norm(s, s['act']).to(TYPES[s['x']])
    return _product(_group_norm(s, 'silu'), s['wq'], s['ws'], None, 'residual', s['res'], 1.0, torch.float32)


# ---------------------------------------------------------------------------- the framework's calls
def _own(s):
    global _runtime
    from parakeet_cuda_b200 import pq8
    from parakeet_cuda_b200.runtime import Int8Weight, Runtime
    if _runtime is None:
        _runtime = Runtime(0)
    rt = _runtime
    epilogues = {'none': pq8.EPI_NONE, 'relu': pq8.EPI_RELU, 'silu': pq8.EPI_SILU, 'glu': pq8.EPI_GLU,
                 'residual': pq8.EPI_RESIDUAL}
    if s['op'] == 'linear':
        return rt.linear_i8(s['x_t'], Int8Weight(s['wq'], s['ws']), bias=s['b'], resid=s['res'],
                            epilogue=epilogues[s['epi']], alpha=0.5,
                            norm=(s['gamma'], s['beta']) if s['norm'] else None, out_dtype=TYPES[s['y']])
    if s['op'] == 'group_norm':
        return rt.group_norm(s['x_t'], s['gamma'], s['beta'], s['groups'], windows=s['windows'],
                             offsets=s['offsets'], epilogue=epilogues[s['act']])
    h = rt.group_norm_quantize(s['x_t'], s['gamma'], s['beta'], s['groups'], windows=s['windows'],
                               offsets=s['offsets'], epilogue=pq8.EPI_SILU)
    return rt.linear_i8(h, Int8Weight(s['wq'], s['ws']), resid=s['res'], epilogue=pq8.EPI_RESIDUAL,
                        out_dtype=torch.float32)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------- work
def work(case):
    size = {'f32': 4, 'f16': 2, 'bf16': 2}
    if case['op'] == 'linear':
        m, k, n = case['m'], case['k'], case['n']
        out = n // 2 if case['epi'] == 'glu' else n
        b = m * k * size[case['x']] + n * k + 4 * n + m * out * size[case['y']]
        b += 4 * n if case['bias'] else 0
        b += m * out * size[case['y']] if case['epi'] == 'residual' else 0
        b += 8 * k if case['norm'] else 0
        return {'bytes': b, 'flops': 2 * m * n * k + (10 if case['norm'] else 2) * m * k}
    rows, c = case['windows'] * case['t'], case['channels']
    extra = 4 * (case['windows'] + 1) if case['ragged'] else 0
    if case['op'] == 'group_norm':
        return {'bytes': 2 * rows * c * size[case['x']] + 8 * c + extra, 'flops': 12 * rows * c}
    n = case['n']
    return {'bytes': rows * c * size[case['x']] + 8 * c + extra + n * c + 4 * n + 8 * rows * n,
            'flops': 14 * rows * c + 2 * rows * c * n}


# ---------------------------------------------------------------------------- definition in 64 bits
def _exact_tokens(h):
    """Scales and integers of rows: the integer whose distance to the quotient is least, the even one of two."""
    top = torch.max(h.max(1).values, -h.min(1).values)
    scale = torch.div(top, 127.0).to(torch.float32).to(torch.float64)
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    u = h / safe[:, None]
    low = torch.floor(u)
    rest = u - low
    odd = torch.remainder(low, 2) == 1
    return low + ((rest > 0.5) | ((rest == 0.5) & odd)).to(torch.float64), scale


def _exact_product(h, wq, ws, bias, epi, res, alpha):
    q, scale = _exact_tokens(h)
    z = torch.nn.functional.linear(q, wq.to(torch.float64))
    z *= ws.to(torch.float64)
    z *= scale[:, None]
    if bias is not None:
        z += bias.to(torch.float64)
    if epi == 'glu':
        a, gate = z.chunk(2, dim=1)
        return a * torch.special.expit(gate)
    if epi == 'silu':
        return z * torch.special.expit(z)
    if epi == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z))
    if epi == 'residual':
        return res.to(torch.float64) + z * alpha
    return z


def _exact_group_norm(s, act):
    x = s['x_t'].to(torch.float64)
    rows, c = x.shape
    step = c // s['groups']
    out = torch.empty_like(x)
    bounds = s['offsets'].tolist() if s['offsets'] is not None else [i * s['t'] for i in range(s['windows'] + 1)]
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        if hi == lo:
            continue
        block = x[lo:hi].unflatten(1, (s['groups'], step))
        var, mean = torch.var_mean(block, dim=(0, 2), correction=0, keepdim=True)
        out[lo:hi] = ((block - mean) / torch.sqrt(var + EPS)).flatten(1)
    out = out * s['gamma'].to(torch.float64) + s['beta'].to(torch.float64)
    return out * torch.special.expit(out) if act == 'silu' else torch.relu(out) if act == 'relu' else out


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'group_norm':
        return _exact_group_norm(s, case['act'])
    if case['op'] == 'norm_linear':
        return _exact_product(_exact_group_norm(s, 'silu'), s['wq'], s['ws'], None, 'residual', s['res'], 1.0)
    h = s['x_t'].to(torch.float64)
    if case['norm']:
        var, mean = torch.var_mean(h, dim=1, correction=0, keepdim=True)
        h = (h - mean) / torch.sqrt(var + EPS) * s['gamma'].to(torch.float64) + s['beta'].to(torch.float64)
    return _exact_product(h, s['wq'], s['ws'], s['b'], case['epi'], s['res'], 0.5)
