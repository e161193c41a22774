"""Cases that measure the 8-bit products and the distillation operators of the recogniser's class layer.

A recogniser (the teacher, float32) is followed by one whose dense layers multiply 8-bit floating point blocks (the
student): activations and weights are quantised in blocks of 128 with a power-of-two scale, multiplied, the student's
logits are compared with the teacher's K largest ones, and the gradient of that loss goes back through the same product.
"""
import torch

own = False

E4M3_MAX = 448.0
BLOCK = 128


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # activations in front of a recogniser's Dense layer: both directions of a BiLSTM of 256 units, 2000 words
        {'name': 'quantise activations', 'op': 'quantise', 'rows': 131072, 'cols': 512, 'dtype': 'bf16', 'block_rows': 1, 'transpose': False},
        # gradient of the logits, transposed: an operand of the class layer's weight gradient
        {'name': 'quantise gradient, transposed', 'op': 'quantise', 'rows': 16384, 'cols': 6719, 'dtype': 'f32', 'block_rows': 1, 'transpose': True},
        # class layer for a single time step
        {'name': 'linear, one step', 'op': 'linear', 'm': 1, 'n': 6719, 'k': 256, 'dtype': 'bf16', 'out': 'f32'},
        # class layer of the english recogniser for one word (63 steps of a crop 256 wide)
        {'name': 'product, one word', 'op': 'product', 'm': 63, 'n': 97, 'k': 256, 'block_rows': 128, 'bias': True, 'out': 'f32'},
        # class layer of the simplified chinese recogniser for the words of a page
        {'name': 'product, class layer', 'op': 'product', 'm': 16384, 'n': 6719, 'k': 256, 'block_rows': 128, 'bias': True, 'out': 'f32'},
        # its weight gradient: both operands in rows of 1 x 128 blocks along the time steps
        {'name': 'product, weight gradient', 'op': 'product', 'm': 6719, 'n': 256, 'k': 16384, 'block_rows': 1, 'bias': False, 'out': 'f32'},
        # a large dense layer
        {'name': 'product, large', 'op': 'product', 'm': 8192, 'n': 8192, 'k': 8192, 'block_rows': 128, 'bias': False, 'out': 'bf16'},
        # teacher's logits of one word
        {'name': 'top logits, one word', 'op': 'top', 'rows': 63, 'v': 97, 'k': 10, 'dtype': 'f32', 'temperature': 1.0},
        # teacher's logits of a page of chinese words
        {'name': 'top logits, page', 'op': 'top', 'rows': 16384, 'v': 6719, 'k': 32, 'dtype': 'f32', 'temperature': 2.0},
        # training batch of the english recogniser: loss and gradient
        {'name': 'distillation, english batch', 'op': 'distil', 'rows': 131072, 'v': 97, 'k': 10, 'dtype': 'f32', 'temperature': 1.0,
         'rest': False, 'grad': True, 'weighted': True},
        # training batch of the chinese recogniser, bfloat16 logits, classes outside the teacher's entries as one
        {'name': 'distillation, chinese batch', 'op': 'distil', 'rows': 16384, 'v': 6719, 'k': 32, 'dtype': 'bf16', 'temperature': 2.0,
         'rest': True, 'grad': True, 'weighted': True},
        # the loss alone over a large vocabulary of odd size
        {'name': 'distillation, large vocabulary', 'op': 'distil', 'rows': 2048, 'v': 131071, 'k': 64, 'dtype': 'bf16', 'temperature': 1.0,
         'rest': True, 'grad': False, 'weighted': False},
    ]


def _spread(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(['quantise', 'linear', 'product', 'product', 'top', 'distil', 'distil'])
    if op == 'quantise':
        rows, cols = _spread(rng, 17, 131072), _spread(rng, 33, 8192)
        rows = max(1, min(rows, (1 << 27) // cols))
        return {'op': op, 'rows': rows, 'cols': cols, 'dtype': rng.choice(['f32', 'bf16']), 'block_rows': rng.choice([1, 128]),
                'transpose': rng.random() < 0.5}
    if op == 'linear':
        return {'op': op, 'm': _spread(rng, 1, 64), 'n': _spread(rng, 64, 8192), 'k': _spread(rng, 64, 8192),
                'dtype': rng.choice(['f32', 'bf16']), 'out': rng.choice(['f32', 'bf16'])}
    if op == 'product':
        m, n, k = _spread(rng, 1, 65536), _spread(rng, 64, 8192), _spread(rng, 64, 16384)
        m = max(1, min(m, int(4e11 // (n * k)), (1 << 28) // n, (1 << 28) // k))
        return {'op': op, 'm': m, 'n': n, 'k': k, 'block_rows': rng.choice([1, 128]), 'bias': rng.random() < 0.5,
                'out': rng.choice(['f32', 'bf16'])}
    v = _spread(rng, 65, 131072)
    rows = max(1, min(_spread(rng, 1, 131072), (1 << 27) // v))
    case = {'op': op, 'rows': rows, 'v': v, 'k': _spread(rng, 1, 64), 'dtype': rng.choice(['f32', 'bf16']),
            'temperature': rng.choice([1.0, 2.0, 4.0])}
    if op == 'distil':
        case.update(rest=rng.random() < 0.5, grad=rng.random() < 0.7, weighted=rng.random() < 0.5)
    return case


def _dtype(name):
    return {'f32': torch.float32, 'bf16': torch.bfloat16}[name]


def _up(n, to):
    return (n + to - 1) // to * to


def work(case):
    size = {'f32': 4, 'bf16': 2}
    if case['op'] == 'quantise':
        n = case['rows'] * case['cols']
        rows, cols = (case['cols'], case['rows']) if case['transpose'] else (case['rows'], case['cols'])
        blocks = -(-rows // case['block_rows']) * -(-cols // BLOCK)
        return {'bytes': n * (size[case['dtype']] + 1) + blocks, 'flops': 2 * n}
    if case['op'] in ('linear', 'product'):
        m, n, k = case['m'], case['n'], case['k']
        a = m * k * size[case['dtype']] if case['op'] == 'linear' else m * k + m * -(-k // BLOCK)
        b_rows = case.get('block_rows', 128)
        b = n * k + -(-n // b_rows) * -(-k // BLOCK)
        return {'bytes': a + b + m * n * size[case['out']] + (4 * n if case.get('bias', True) else 0), 'flops': 2 * m * n * k}
    rows, v, k = case['rows'], case['v'], min(case['k'], case['v'])
    read = rows * v * size[case['dtype']]
    if case['op'] == 'top':
        return {'bytes': read + rows * (8 * k + 4), 'flops': 4 * rows * v}
    return {'bytes': read * (2 if case['grad'] else 1) + rows * (8 * k + 4 + (4 if case['rest'] else 0) + (4 if case['weighted'] else 0)),
            'flops': (6 if case['grad'] else 4) * rows * v}


# -------------------------------------------------------------------------------------------- inputs
def _activations(g, rows, cols):
    """Values of a layer's output: columns of different scale, a few large ones, and blocks of zeros."""
    x = torch.randn(rows, cols, generator=g, device='cuda')
    x *= torch.exp2(torch.randint(-3, 4, (cols,), generator=g, device='cuda').float())
    x[torch.rand(rows, generator=g, device='cuda') < 0.01] = 0.0
    return x


def _blocks(x, block_rows):
    """(rows, cols) -> (row blocks, block_rows, column blocks, 128), padded with zeros."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, _up(cols, BLOCK) - cols, 0, _up(rows, block_rows) - rows))
    return x.reshape(-1, block_rows, x.shape[1] // BLOCK, BLOCK)


def _scale_exponent(amax):
    """Least e with amax <= 448 * 2^e, 0 for a block of zeros, at least -127."""
    m, e = torch.frexp(amax)                                  # amax = m * 2^e, 0.5 <= m < 1
    return torch.where(amax == 0, 0, torch.clamp(e - 9 + (m > 0.875).to(e.dtype), min=-127))


def _quantise(x, block_rows):
    """-> (bytes as float8 (rows, cols rounded up to 128), exponents + 127 as uint8 (column blocks, row blocks))"""
    rows = x.shape[0]
    b = _blocks(x.float(), block_rows)
    e = _scale_exponent(b.abs().amax(dim=(1, 3), keepdim=True))
    half = torch.div(e, 2, rounding_mode='floor')              # two factors: 2^127 and beyond is no float32
    q = (b * torch.exp2(-half.float()) * torch.exp2(-(e - half).float())).to(torch.float8_e4m3fn)
    q = q.reshape(-1, b.shape[2] * BLOCK)[:rows].contiguous()
    return q, (e[:, 0, :, 0] + 127).to(torch.uint8).t().contiguous()


def _operand(g, rows, cols, block_rows, scale=1.0):
    q, e = _quantise(_activations(g, rows, cols) * scale, block_rows)
    lead = _up(e.shape[1], 16)                                 # rows of the scale table start on 16 bytes
    table = torch.full((e.shape[0], lead), 127, dtype=torch.uint8, device='cuda')
    table[:, :e.shape[1]] = e
    return {'q': q, 'scale': table, 'rows': rows, 'cols': cols, 'block_rows': block_rows}


def _logits(g, rows, v):
    """Logits of a recogniser: noise, one class far above the others in most steps, the first class (blank) in many."""
    x = torch.randn(rows, v, generator=g, device='cuda') * 2.0
    top = torch.randint(0, v, (rows, 1), generator=g, device='cuda')
    top = torch.where(torch.rand(rows, 1, generator=g, device='cuda') < 0.4, 0, top)
    x.scatter_add_(1, top, torch.rand(rows, 1, generator=g, device='cuda') * 12.0)
    return x


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    op, state = case['op'], dict(case)
    if op == 'quantise':
        state['x'] = _activations(g, case['rows'], case['cols']).to(_dtype(case['dtype']))
    elif op in ('linear', 'product'):
        m, n, k = case['m'], case['n'], case['k']
        state['w'] = _operand(g, n, k, case.get('block_rows', 128), k ** -0.5)
        if op == 'linear':
            state['x'] = _activations(g, m, k).to(_dtype(case['dtype']))
        else:
            state['a'] = _operand(g, m, k, 1)
        state['b'] = torch.randn(n, generator=g, device='cuda') if case.get('bias', True) else None
    else:
        rows, v, k = case['rows'], case['v'], min(case['k'], case['v'])
        teacher = _logits(g, rows, v)
        if op == 'top':
            state['x'] = teacher.to(_dtype(case['dtype']))
        else:
            t = case['temperature']
            values, index = torch.topk(teacher, k)
            state['values'], state['index'] = values.contiguous(), index.to(torch.int32)
            state['lse'] = torch.logsumexp(teacher / t, 1) if case['rest'] else None
            state['x'] = (teacher + 0.7 * torch.randn(rows, v, generator=g, device='cuda')).to(_dtype(case['dtype']))
            # rows with fewer entries than the table is wide, and rows without any
            few = torch.rand(rows, 1, generator=g, device='cuda')
            keep = torch.arange(k, device='cuda') < torch.where(few < 0.01, 0.0, torch.where(few < 0.1, k / 2.0, float(k)))
            state['index'] = torch.where(keep, state['index'], -1).contiguous()
            # steps behind the end of a sequence in a padded batch carry no weight
            state['weight'] = (torch.rand(rows, generator=g, device='cuda') > 0.1).float() / rows if case['weighted'] else None
    return state


# ----------------------------------------------------------------------------------------- plain form
def _dequantise(q, scale, rows, cols, block_rows):
    e = scale[:, :-(-rows // block_rows)].t().to(torch.float32) - 127.0
    e = e.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)
    return (q.float() * torch.exp2(e))[:, :cols]


def _product(a, w, bias, out):
    c = _dequantise(**a) @ _dequantise(**w).t()
    return (c if bias is None else c + bias).to(_dtype(out))


def _top(x, k, temperature):
    x = x.float()
    values, index = torch.sort(x, dim=1, descending=True, stable=True)
    high = values[:, :1]
    lse = torch.log(torch.exp((x - high) / temperature).sum(1)) + high[:, 0] / temperature
    return {'values': values[:, :k].contiguous(), 'index': index[:, :k].to(torch.int32), 'lse': lse}


def _distil(x, values, index, lse, temperature, weight, grad):
    """The sums over the classes outside the teacher's entries in 32 bits; the few numbers of a row that the loss is a
    difference of (where teacher and student nearly agree it is far smaller than its terms) in 64."""
    rows, v = x.shape
    t = temperature
    there = index >= 0
    at = torch.where(there, index, 0).long()
    inside = torch.zeros(rows, v + 1, dtype=torch.bool, device=x.device)
    inside.scatter_(1, torch.where(there, index, v).long(), True)
    inside = inside[:, :v]
    s = x.float()
    high = s.amax(1, keepdim=True)
    e = torch.exp((s - high) / t)
    rest = torch.where(inside, 0.0, e).sum(1, dtype=torch.float64)
    s_k = (torch.gather(s, 1, at).double() - high) / t
    again = ((index[:, :, None] == index[:, None, :]).tril(-1)).any(2)        # an entry that names a class a second time
    total = rest + torch.where(there & ~again, torch.exp(s_k), 0.0).sum(1)
    log_q = s_k - torch.log(total)[:, None]
    z = torch.where(there, values.double() / t, -torch.inf)
    if lse is None:
        top = z.amax(1, keepdim=True)
        top = torch.where(torch.isfinite(top), top, 0.0)
        sum_p = torch.exp(z - top).sum(1, keepdim=True)
        log_p = z - top - torch.log(torch.where(sum_p > 0, sum_p, 1.0))
    else:
        log_p = z - lse[:, None].double()
    p = torch.exp(log_p)
    loss = torch.where(p > 0, p * (torch.where(p > 0, log_p, 0.0) - log_q), 0.0).sum(1)
    if lse is not None:
        p_rest = torch.clamp(1.0 - p.sum(1), min=0.0)
        loss = loss + torch.where(p_rest > 0, p_rest * (torch.log(torch.where(p_rest > 0, p_rest, 1.0)) - torch.log(rest / total)), 0.0)
    scale = torch.ones(rows, device=x.device) if weight is None else weight
    out = {'loss': (loss * scale * (t * t)).float()}
    if grad:
        outside = 1.0 / total if lse is None else 1.0 / total - p_rest / rest
        g = e * torch.where(there.any(1), outside, 0.0 if lse is None else outside).float()[:, None]
        q_k = torch.exp(log_q) if lse is not None else torch.where(there.any(1, keepdim=True), torch.exp(log_q), 0.0)
        same = (index[:, :, None] == index[:, None, :]) & there[:, None, :]
        g_k = (q_k - torch.where(same, p[:, None, :], 0.0).sum(2)).float()
        g = torch.cat([g, g.new_zeros(rows, 1)], 1).scatter_(1, torch.where(there, index, v).long(), g_k)[:, :v]
        out['grad'] = (g * (scale * t)[:, None]).to(x.dtype)
    return out


_kept = {}


def _context():
    """The handle that a program creates once."""
    if 'ctx' not in _kept:
        from ocr_amd.engine import HipContext
        _kept['ctx'] = HipContext(torch.cuda.current_device())
    return _kept['ctx']


def _own(state):
    from ocr_amd.engine import Fp8Matrix
    ctx, op = _context(), state['op']
    if op == 'quantise':
        m = ctx.quantize_fp8(state['x'], block_rows=state['block_rows'], transpose=state['transpose'])
        return {'q': m.q, 'scale': m.scale[:, :-(-m.rows // m.block_rows)]}
    if op == 'linear':
        return ctx.linear_fp8(state['x'], Fp8Matrix(**state['w']), bias=state['b'], out_dtype=_dtype(state['out']))
    if op == 'product':
        return ctx.gemm_fp8(Fp8Matrix(**state['a']), Fp8Matrix(**state['w']), bias=state['b'], out_dtype=_dtype(state['out']))
    if op == 'top':
        values, index, lse = ctx.top_logits(state['x'], min(state['k'], state['v']), temperature=state['temperature'])
        return {'values': values, 'index': index, 'lse': lse}
    out = ctx.distill_loss(state['x'], state['values'], state['index'], top_lse=state['lse'], temperature=state['temperature'],
                           row_weight=state['weight'], want_grad=state['grad'])
    return {k: out[k] for k in (('loss', 'grad') if state['grad'] else ('loss',))}


def run(state):
    if own:
        return _own(state)
    op = state['op']
    if op == 'quantise':
        q, e = _quantise(state['x'].t() if state['transpose'] else state['x'], state['block_rows'])
        return {'q': q, 'scale': e}
    if op == 'linear':
        q, e = _quantise(state['x'], 1)
        return _product({'q': q, 'scale': e, 'rows': state['m'], 'cols': state['k'], 'block_rows': 1}, state['w'], state['b'], state['out'])
    if op == 'product':
        return _product(state['a'], state['w'], state['b'], state['out'])
    if op == 'top':
        return _top(state['x'], min(state['k'], state['v']), state['temperature'])
    return _distil(state['x'], state['values'], state['index'], state['lse'], state['temperature'], state['weight'], state['grad'])


# --------------------------------------------------------------------------------- 64-bit definition
def _e4m3_64(x):
    """float64 -> the nearest e4m3 value (ties to the even mantissa), |x| <= 448: three bits behind the leading one,
    exponents from -6 on, steps of 2^-9 below."""
    m, e = torch.frexp(x)
    step = torch.exp2(torch.clamp(e.double() - 4, min=-9))
    return torch.round(x / step) * step                       # torch.round takes halves to the even multiple


def _blocks_64(x, block_rows):
    """float64 matrix -> (e4m3 values, exponents) by the definition, for all blocks at once."""
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    full = torch.zeros(rb * block_rows, cb * BLOCK, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    amax = full.abs().view(rb, block_rows, cb, BLOCK).amax(3).amax(1)
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, E4M3_MAX) / E4M3_MAX))
    e = torch.where(amax > E4M3_MAX * torch.exp2(e), e + 1, e)                    # log2's own rounding
    e = torch.where((amax > 0) & (amax <= E4M3_MAX * torch.exp2(e - 1)), e - 1, e).clamp(min=-127)
    by = torch.exp2(e).repeat_interleave(block_rows, 0).repeat_interleave(BLOCK, 1)
    return _e4m3_64(full / by)[:rows], e, by[:rows]


def _values_64(m):
    rows, cols, by = m['rows'], m['cols'], m['block_rows']
    e = m['scale'].double()[:, :-(-rows // by)].t() - 127
    row = torch.arange(rows, device=e.device) // by
    col = torch.arange(cols, device=e.device) // BLOCK
    return m['q'].double()[:, :cols] * torch.exp2(e[row][:, col])


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op == 'quantise':
        x = s['x'].double()
        q, e, _ = _blocks_64(x.t().contiguous() if case['transpose'] else x, case['block_rows'])
        return {'q': q, 'scale': None}
    if op in ('linear', 'product'):
        if op == 'linear':
            q, _, by = _blocks_64(s['x'].double(), 1)
            a = (q * by)[:, :case['k']]
        else:
            a = _values_64(s['a'])
        c = torch.matmul(a, _values_64(s['w']).t().contiguous())
        return c if s['b'] is None else c + s['b'].double()
    x, t = s['x'].double(), case['temperature']
    if op == 'top':
        k = min(case['k'], case['v'])
        return {'values': torch.topk(x, k).values, 'index': None, 'lse': torch.logsumexp(x / t, 1)}
    log_q = torch.log_softmax(x / t, 1)
    there = s['index'] >= 0
    at = s['index'].clamp(min=0).long()
    z = torch.where(there, s['values'].double() / t, -torch.inf)
    if case['rest']:
        p = torch.exp(z - s['lse'].double()[:, None])
    else:
        p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
    inside = torch.zeros_like(log_q)
    inside.scatter_add_(1, at, there.double())
    target = torch.zeros_like(log_q).scatter_add_(1, at, torch.where(there, p, 0.0))
    loss = (torch.special.xlogy(p, p) - torch.where(there, p * torch.gather(log_q, 1, at), 0.0)).sum(1)
    q = torch.exp(log_q)
    if case['rest']:
        p_rest = (1.0 - p.sum(1)).clamp(min=0.0)
        log_rest = torch.logsumexp(torch.where(inside > 0, -torch.inf, log_q), 1)
        loss = loss + torch.special.xlogy(p_rest, p_rest) - torch.where(p_rest > 0, p_rest * log_rest, 0.0)
        target = torch.where(inside > 0, target, p_rest[:, None] * torch.exp(log_q - log_rest[:, None]))
        grad = q - target
    else:
        grad = torch.where(there.any(1, keepdim=True), q - target, 0.0)
    w = torch.ones(case['rows'], dtype=torch.float64, device=x.device) if s['weight'] is None else s['weight'].double()
    out = {'loss': loss * w * t * t}
    if case['grad']:
        out['grad'] = grad * (w * t)[:, None]
    return out
