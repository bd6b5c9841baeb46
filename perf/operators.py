"""Cases for the matrix products that read quantized tensors, for the products grouped by expert, and for the NVFP4 cast.

Four operators, named by a case's `op`:

  nvfp4     quant.per_token_cast_to_nvfp4 and quant.cast_back: FP4 codes with an e4m3 scale per 16 values and one fp32
            scale per tensor, and the way back
  dense     quant.block_scaled_gemm: out = alpha * a @ b.T for two quantized matrices
  grouped   moe.grouped_gemm: rows sorted by expert times each expert's weight (bf16 or quantized); with `transpose` the
            product with the transposed weight, which is the gradient of the rows
  wgrad     moe.grouped_gemm_wgrad: the gradient of each expert's weight

Quantized operands (`fmt`): "fp8_128" is e4m3 with a power-of-two scale per 128 values of an activation row and per
128 x 128 block of a weight, "fp8_32" e4m3 with one per 32 values of a row (both operands), "mxfp4" e2m1 with one per 32
values, "nvfp4" e2m1 with an e4m3 scale per 16 values and a scale per tensor.  Power-of-two scales are packed four to an
int32 word, column-major, as the casts write them.

The widths 7168 and 2048 (4096 for gate and up together) are the ones of this repository's own benchmark.
"""
import math
import random

import torch

own = False

E4M3_MAX, E2M1_MAX = 448.0, 6.0
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_FMTS = ('fp8_128', 'fp8_32', 'mxfp4', 'nvfp4')


def listed():
    return [
        # one token's activations on the way into a 4-bit layer: launch latency
        dict(name='nvfp4_token', op='nvfp4', rows=1, hidden=7168, dtype='bf16'),
        # a prefill batch of an odd number of tokens: memory bandwidth
        dict(name='nvfp4_prefill', op='nvfp4', rows=20001, hidden=7168, dtype='bf16'),
        # the gate-and-up projection of a large prefill batch in 4 bits
        dict(name='dense_mxfp4_prefill', op='dense', fmt='mxfp4', m=16384, n=4096, k=7168),
        # the down projection of a batch of odd length
        dict(name='dense_nvfp4_odd', op='dense', fmt='nvfp4', m=4001, n=7168, k=2048),
        # one token through an FP8 layer: the weight's bytes and the latency are all there is
        dict(name='dense_fp8_token', op='dense', fmt='fp8_128', m=1, n=4096, k=7168),
        # gate-and-up projection of the experts in a prefill, expert segments aligned to 128 rows by the expansion
        dict(name='grouped_fp8_prefill', op='grouped', fmt='fp8_128', experts=32, rows=16384, spare=4096, align=128, n=4096, k=7168, transpose=False),
        # the same layer in 4 bits while decoding a small batch: a few rows per expert, some experts without any
        dict(name='grouped_mxfp4_decode', op='grouped', fmt='mxfp4', experts=32, rows=61, spare=3, align=1, n=4096, k=7168, transpose=False),
        # down projection of a chunk, segments of any length
        dict(name='grouped_nvfp4_chunk', op='grouped', fmt='nvfp4', experts=16, rows=3989, spare=0, align=1, n=7168, k=2048, transpose=False),
        # a training step of the experts: forward, gradient of the rows, gradient of the weights
        dict(name='grouped_bf16_forward', op='grouped', fmt='bf16', experts=16, rows=8192, spare=256, align=16, n=4096, k=7168, transpose=False),
        dict(name='grouped_bf16_dgrad', op='grouped', fmt='bf16', experts=16, rows=8192, spare=256, align=16, n=7168, k=4096, transpose=True),
        dict(name='wgrad_fp32', op='wgrad', experts=16, rows=8192, spare=256, align=16, n=4096, k=7168, out='fp32'),
        # a small layer with few tokens per expert, odd sizes
        dict(name='wgrad_bf16_small', op='wgrad', experts=8, rows=777, spare=5, align=1, n=1032, k=2056, out='bf16'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('nvfp4', 'dense', 'dense', 'grouped', 'grouped', 'grouped', 'wgrad', 'wgrad'))
    if op == 'nvfp4':
        hidden = 64 * _log(rng, 4, 128)
        rows = min(_log(rng, 1, 40000), 20000 * 7168 // hidden)
        return dict(op=op, rows=rows, hidden=hidden, dtype=rng.choice(('bf16', 'bf16', 'fp32')))
    limit = 16384 * 4096 * 7168
    n = 8 * _log(rng, 16, 1024)
    if op == 'dense':
        k = 64 * _log(rng, 4, 128)
        return dict(op=op, fmt=rng.choice(_FMTS), m=min(_log(rng, 1, 20000), limit // (n * k)), n=n, k=k)
    experts = _log(rng, 1, 64)
    align = rng.choice((1, 1, 16, 128))
    if op == 'grouped':
        transpose = rng.random() < 0.25
        fmt = 'bf16' if transpose or rng.random() < 0.25 else rng.choice(_FMTS)
        k = (8 * _log(rng, 16, 1024)) if fmt == 'bf16' else 64 * _log(rng, 4, 128)
        n, k = _within(experts, n, k)
        rows = max(1, min(_log(rng, 1, 20000), limit // (n * k)))
        return dict(op=op, fmt=fmt, experts=experts, rows=rows, spare=rng.randrange(0, 65), align=align, n=n, k=k, transpose=transpose)
    n, k = _within(experts, n, 8 * _log(rng, 16, 1024))
    rows = max(1, min(_log(rng, 1, 20000), limit // (n * k)))
    return dict(op=op, experts=experts, rows=rows, spare=rng.randrange(0, 65), align=align, n=n, k=k, out=rng.choice(('fp32', 'bf16')))


def _within(experts, n, k):
    """Weights of at most 32 x 4096 x 7168 values."""
    while experts * n * k > 32 * 4096 * 7168:
        n, k = max(128, n // 128 * 64), max(256, k // 128 * 64)
    return n, k


# --- formats, in plain operations ----------------------------------------------------------------------------------


def _e2m1_code(v):
    """Code of the nearest e2m1 value, ties to the even code."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8)
    c += a >= 0.75
    c += a > 1.25
    c += a >= 1.75
    c += a > 2.5
    c += a >= 3.5
    c += a > 5.0
    return c | (torch.signbit(v).to(torch.uint8) << 3)


def _pack_codes(c):
    return (c[..., 0::2] | (c[..., 1::2] << 4)).view(torch.int8)


def _unpack_codes(q, dtype):
    u = q.view(torch.uint8)
    table = torch.tensor(_E2M1, dtype=dtype, device=q.device)
    return table[torch.stack((u & 15, u >> 4), dim=-1).flatten(-2).to(torch.int32)]


def _e4m3(r):
    """Nearest e4m3 number of r >= 0 (64 bits), ties to even: three mantissa bits, none finer than 2^-9."""
    step = torch.exp2((torch.frexp(r).exponent - 1).clamp(min=-6).double() - 3)
    return (torch.round(r / step) * step).to(torch.float8_e4m3fn)


def _pow2_scale(amax, top):
    """Biased exponent of the smallest power of two that is not below amax / top."""
    bits = (amax.clamp(min=1e-4) / top).view(torch.int32)
    return ((bits - 1) >> 23) + 1


def _pack_exponents(e):
    """(rows, groups) exponent bytes -> (rows, words) int32, column-major with the rows padded to four."""
    rows, groups = e.shape
    words, pitch = -(-groups // 4), -(-rows // 4) * 4
    store = torch.zeros((words, pitch, 4), dtype=torch.uint8, device=e.device)
    full = torch.zeros((rows, words * 4), dtype=torch.uint8, device=e.device)
    full[:, :groups] = e
    store[:, :rows] = full.view(rows, words, 4).permute(1, 0, 2)
    return store.view(torch.int32).view(words, pitch).T[:rows]


def _unpack_exponents(words, groups):
    return (words[..., None] >> torch.arange(0, 32, 8, device=words.device) & 255).flatten(-2)[..., :groups]


def _quantize(x, fmt, weight, ts=None):
    """What the casts make of x (2-D, fp32): (codes, scales)."""
    rows, k = x.shape
    if fmt == 'nvfp4':
        # in 64 bits: the borders between codes are met often (a block's values are ratios of short numbers)
        g, ts = x.double().view(rows, k // 16, 16), ts.double()
        sf = _e4m3((g.abs().amax(dim=-1) / (E2M1_MAX * ts)).clamp(max=E4M3_MAX))
        d = (sf.double() * ts)[..., None]
        return _pack_codes(_e2m1_code(torch.where(d > 0, g / d, 0.0).view(rows, k))), sf
    group = {'fp8_128': 128, 'fp8_32': 32, 'mxfp4': 32}[fmt]
    top = E2M1_MAX if fmt == 'mxfp4' else E4M3_MAX
    pad = torch.nn.functional.pad(x, (0, -k % group))
    amax = pad.view(rows, -1, group).abs().amax(dim=-1)
    if fmt == 'fp8_128' and weight:
        blocks = torch.nn.functional.pad(amax, (0, 0, 0, -rows % 128)).view(-1, 128, amax.shape[1]).amax(dim=1)
        e = _pow2_scale(blocks, top)
        per_row = e.repeat_interleave(128, 0)[:rows]
    else:
        e = per_row = _pow2_scale(amax, top)
    inv = ((254 - per_row) << 23).view(torch.float32).repeat_interleave(group, 1)[:, :k]
    v = x * inv
    codes = _pack_codes(_e2m1_code(v)) if fmt == 'mxfp4' else v.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes, _pack_exponents(e)


def _values(q, sf, fmt, rows_per_scale, k, dtype):
    """The numbers a quantized matrix stands for (without the tensor scale)."""
    if fmt == 'nvfp4':
        return _unpack_codes(q, dtype) * sf.to(dtype).repeat_interleave(16, -1)
    group = {'fp8_128': 128, 'fp8_32': 32, 'mxfp4': 32}[fmt]
    v = _unpack_codes(q, dtype) if fmt == 'mxfp4' else q.to(dtype)
    s = torch.exp2(_unpack_exponents(sf, -(-k // group)).to(dtype) - 127)
    s = s.repeat_interleave(rows_per_scale, 0)[:v.shape[0]].repeat_interleave(group, 1)[:, :k]
    return v * s


def _block(fmt, weight):
    return {'fp8_128': (128, 128) if weight else (1, 128), 'fp8_32': (1, 32), 'mxfp4': (1, 32), 'nvfp4': (1, 16), 'bf16': None}[fmt]


# --- inputs --------------------------------------------------------------------------------------------------------


def _activations(gen, rows, cols, outliers=1e-3):
    x = torch.randn((rows, cols), generator=gen, device='cuda')
    if outliers:  # a few channels of a transformer's activations are far larger than the rest
        x[:, torch.rand(cols, generator=gen, device='cuda') < outliers] *= 20
    return x


def _segments(seed, experts, rows, align):
    """Ragged expert segments: skewed sizes that add up to `rows`, each segment's start a multiple of `align`; and the
    rows that any such segments fit in."""
    rng = random.Random(seed)
    weights = [rng.random() ** 2 for _ in range(experts)]
    total = sum(weights) or 1.0
    sizes = [int(rows * w / total) for w in weights]
    for _ in range(rows - sum(sizes)):
        sizes[rng.randrange(experts)] += 1
    start, end, at = [], [], 0
    for size in sizes:
        start.append(at)
        end.append(at + size)
        at = -(-(at + size) // align) * align
    return start, end, rows + experts * (align - 1)


def _operand(gen, fmt, x, weight):
    """A matrix as the program holds it: bf16, or codes with scales and (NVFP4) the tensor scale."""
    if fmt == 'bf16':
        return dict(data=x.to(torch.bfloat16))
    ts = (x.abs().amax() / (E2M1_MAX * E4M3_MAX)).reshape(1) if fmt == 'nvfp4' else None
    q, sf = _quantize(x.to(torch.bfloat16).float(), fmt, weight, ts)
    return dict(data=q, sf=sf, ts=ts)


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    op = case['op']
    if op == 'nvfp4':
        x = _activations(gen, case['rows'], case['hidden']).to(torch.bfloat16 if case['dtype'] == 'bf16' else torch.float32)
        # a calibrated scale: largest magnitude over largest code times largest block scale
        return dict(case=case, x=x, ts=(x.float().abs().amax() / (E2M1_MAX * E4M3_MAX)).reshape(1))
    if op == 'dense':
        a = _operand(gen, case['fmt'], _activations(gen, case['m'], case['k']), False)
        b = _operand(gen, case['fmt'], 0.02 * torch.randn((case['n'], case['k']), generator=gen, device='cuda'), True)
        alpha = a['ts'] * b['ts'] if case['fmt'] == 'nvfp4' else None
        return dict(case=case, a=a, b=b, alpha=alpha)
    experts, n, k = case['experts'], case['n'], case['k']
    start, end, room = _segments(seed, experts, case['rows'], case['align'])
    rows = room + case['spare']
    state = dict(case=case, longest=max(e - s for s, e in zip(start, end)),
                 start=torch.tensor(start, dtype=torch.int32, device='cuda'), end=torch.tensor(end, dtype=torch.int32, device='cuda'))
    # the expansion clears the rows that no token was routed to
    member = torch.zeros(rows, dtype=torch.bool)
    for s, e in zip(start, end):
        member[s:e] = True
    member = member.cuda()[:, None]
    if op == 'wgrad':
        state['x'] = (_activations(gen, rows, k) * member).to(torch.bfloat16)
        state['grad'] = (0.1 * torch.randn((rows, n), generator=gen, device='cuda') * member).to(torch.bfloat16)
        return state
    fmt = case['fmt']
    state['x'] = _operand(gen, fmt, _activations(gen, rows, k) * member, False)
    if fmt == 'bf16':
        shape = (experts, k, n) if case['transpose'] else (experts, n, k)
        state['w'] = dict(data=torch.randn(shape, generator=gen, device='cuda', dtype=torch.bfloat16) * 0.02)
        state['alpha'] = None
        return state
    # every expert's weight is quantized by itself, as a loader does, and kept stacked
    parts, scales = [], []
    for _ in range(experts):
        w = _operand(gen, fmt, 0.02 * torch.randn((n, k), generator=gen, device='cuda'), True)
        parts.append(w['data'])
        scales.append((w['sf'], w['ts']))
    w = dict(data=torch.stack([p.view(torch.uint8) for p in parts]).view(parts[0].dtype))
    if fmt == 'nvfp4':
        w['sf'] = torch.stack([s.view(torch.uint8) for s, _ in scales]).view(torch.float8_e4m3fn)
        state['alpha'] = state['x']['ts'] * torch.cat([t for _, t in scales])
    else:
        w['sf'] = torch.stack([s.T.contiguous() for s, _ in scales]).transpose(1, 2)
        state['alpha'] = None
    state['w'] = w
    return state


# --- one pass ------------------------------------------------------------------------------------------------------


def run(state):
    case = state['case']
    op = case['op']
    if own:
        from tilekernels_b200 import moe, quant
        if op == 'nvfp4':
            q, sf = quant.per_token_cast_to_nvfp4(state['x'], state['ts'])
            return dict(sf=sf, back=quant.cast_back((q, sf), case['dtype'], (1, 16), tensor_scale=state['ts']))
        if op == 'dense':
            a, b, fmt = state['a'], state['b'], case['fmt']
            return quant.block_scaled_gemm((a['data'], a['sf']), (b['data'], b['sf']), _block(fmt, False), _block(fmt, True), alpha=state['alpha'])
        if op == 'wgrad':
            return moe.grouped_gemm_wgrad(state['grad'], state['x'], state['start'], state['end'],
                                          out_dtype=torch.float32 if case['out'] == 'fp32' else torch.bfloat16)
        x, w, fmt = state['x'], state['w'], case['fmt']
        if fmt == 'bf16':
            return moe.grouped_gemm(x['data'], w['data'], state['start'], state['end'], transpose_w=case['transpose'])
        return moe.grouped_gemm((x['data'], x['sf']), (w['data'], w['sf']), state['start'], state['end'], _block(fmt, False), _block(fmt, True),
                                alpha=state['alpha'])
    if op == 'nvfp4':
        x = state['x'].float()
        q, sf = _quantize(x, 'nvfp4', False, state['ts'])
        back = _unpack_codes(q, torch.float64) * (sf.double() * state['ts']).repeat_interleave(16, -1)
        return dict(sf=sf, back=back.to(state['x'].dtype))
    if op == 'dense':
        a, b = _dense_operands(state, torch.float32)
        out = a @ b.T
        return (out if state['alpha'] is None else out * state['alpha']).to(torch.bfloat16)
    rows_of, inside = _padded_rows(state)
    if op == 'wgrad':
        g = state['grad'].float()[rows_of] * inside
        x = state['x'].float()[rows_of] * inside
        return torch.bmm(g.transpose(1, 2), x).to(torch.float32 if case['out'] == 'fp32' else torch.bfloat16)
    x, w = _grouped_operands(state, torch.float32)
    y = torch.bmm(x[rows_of], w if case['transpose'] else w.transpose(1, 2))
    if state['alpha'] is not None:
        y = y * state['alpha'][:, None, None]
    out = torch.zeros((x.shape[0], case['n']), dtype=torch.bfloat16, device=x.device)
    out[rows_of[inside[..., 0]]] = y[inside[..., 0]].to(torch.bfloat16)
    return out


def _padded_rows(state):
    """Row numbers (experts, longest) of every expert's segment, and which of them belong to it."""
    at = state['start'].long()[:, None] + torch.arange(max(1, state['longest']), device='cuda')
    inside = at < state['end'].long()[:, None]
    return torch.where(inside, at, 0), inside[..., None]


def _dense_operands(state, dtype):
    case, a, b = state['case'], state['a'], state['b']
    fmt, k = case['fmt'], case['k']
    return _values(a['data'], a['sf'], fmt, 1, k, dtype), _values(b['data'], b['sf'], fmt, _block(fmt, True)[0], k, dtype)


def _grouped_operands(state, dtype):
    case, x, w = state['case'], state['x'], state['w']
    fmt, k = case['fmt'], case['k']
    if fmt == 'bf16':
        return x['data'].to(dtype), w['data'].to(dtype)
    experts, n = w['data'].shape[:2]
    xv = _values(x['data'], x['sf'], fmt, 1, k, dtype)
    if fmt == 'nvfp4':
        return xv, _values(w['data'], w['sf'], fmt, 1, k, dtype)
    group, block = (128, 128) if fmt == 'fp8_128' else (32, 1)
    v = _unpack_codes(w['data'], dtype) if fmt == 'mxfp4' else w['data'].to(dtype)
    e = _unpack_exponents(w['sf'], -(-k // group))
    s = torch.exp2(e.to(dtype) - 127).repeat_interleave(block, 1)[:, :n].repeat_interleave(group, 2)[..., :k]
    return xv, v * s


def work(case):
    op = case['op']
    if op == 'nvfp4':
        values, width = case['rows'] * case['hidden'], 2 if case['dtype'] == 'bf16' else 4
        # the cast reads x and writes codes and scales, the way back reads those and writes the values
        return dict(bytes=values * (2 * width) + 2 * (values // 2 + values // 16), flops=4 * values)
    per_value = {'bf16': 2.0, 'fp8_128': 1.0 + 1 / 128, 'fp8_32': 1.0 + 1 / 32, 'mxfp4': 0.5 + 1 / 32, 'nvfp4': 0.5 + 1 / 16}
    if op == 'dense':
        m, n, k, b = case['m'], case['n'], case['k'], per_value[case['fmt']]
        return dict(bytes=int((m + n) * k * b + 2 * m * n), flops=2 * m * n * k)
    experts, rows, n, k = case['experts'], case['rows'], case['n'], case['k']
    if op == 'wgrad':
        return dict(bytes=2 * rows * (n + k) + experts * n * k * (4 if case['out'] == 'fp32' else 2), flops=2 * rows * n * k)
    # an expert without rows need not be read: at most `rows` experts have any
    b = per_value[case['fmt']]
    return dict(bytes=int((rows * k + min(experts, rows) * n * k) * b + 2 * rows * n), flops=2 * rows * n * k)


# --- the definition in 64 bits -------------------------------------------------------------------------------------


def _exact_codes(q):
    """e2m1: sign, two exponent bits (bias 1), one mantissa bit."""
    u = q.view(torch.uint8).to(torch.int16)
    c = torch.stack((u % 16, u // 16), dim=-1).flatten(-2)
    sign, e, m = c // 8, (c // 2) % 4, (c % 2).double()
    v = torch.where(e == 0, m * 0.5, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
    return torch.where(sign == 1, -v, v)


def _exact_matrix(q, sf, fmt, rows, k, weight):
    """One quantized matrix in 64 bits, scale by scale."""
    v = _exact_codes(q) if fmt in ('mxfp4', 'nvfp4') else q.double()
    if fmt == 'nvfp4':
        return (v.view(rows, k // 16, 16) * sf.double()[:, :, None]).view(rows, k)
    group, block = (128, 128 if weight else 1) if fmt == 'fp8_128' else (32, 1)
    col = torch.arange(k, device=q.device) // group
    row = torch.arange(rows, device=q.device) // block
    byte = (sf.long()[row][:, col // 4] >> (8 * (col % 4))) & 255
    return v * torch.exp2((byte - 127).double())


def exact(case, seed):
    state = prepare(case, seed)
    op = case['op']
    if op == 'nvfp4':
        x, ts = state['x'].double(), state['ts'].double()
        g = x.view(case['rows'], -1, 16)
        # the block scale: the number of e4m3's positive values, in order, whose border to the next the ratio has passed
        scales = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
        amax, border = g.abs().amax(-1), (scales[1:] + scales[:-1]) * 3 * ts
        at = torch.bucketize(amax, border)
        at += (amax == border[at.clamp(max=125)]) & (at % 2 == 1) & (at < 126)  # on it: the even one
        sf = scales[at]
        d = (sf * ts)[..., None]
        levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        code = torch.zeros_like(g, dtype=torch.int64)
        for i in range(7):  # past the middle of two levels, or on it with an even code above: the products are exact
            middle = (levels[i] + levels[i + 1]) / 2 * d
            code += ((g.abs() > middle) | ((g.abs() == middle) & (i % 2 == 1))) & (d > 0)
        return dict(sf=sf, back=(levels[code] * torch.sign(g) * d).view(x.shape))
    if op == 'dense':
        m, n, k, fmt = case['m'], case['n'], case['k'], case['fmt']
        a = _exact_matrix(state['a']['data'], state['a']['sf'], fmt, m, k, False)
        b = _exact_matrix(state['b']['data'], state['b']['sf'], fmt, n, k, True)
        return (a @ b.T) * (1.0 if state['alpha'] is None else state['alpha'].double())
    spans = list(zip(state['start'].tolist(), state['end'].tolist()))
    if op == 'wgrad':
        out = torch.zeros((case['experts'], case['n'], case['k']), dtype=torch.float64, device='cuda')
        for e, (s, t) in enumerate(spans):
            out[e] = state['grad'][s:t].double().T @ state['x'][s:t].double()
        return out
    fmt, n, k = case['fmt'], case['n'], case['k']
    rows = state['x']['data'].shape[0]
    out = torch.zeros((rows, n), dtype=torch.float64, device='cuda')
    x = state['x']['data'].double() if fmt == 'bf16' else _exact_matrix(state['x']['data'], state['x']['sf'], fmt, rows, k, False)
    for e, (s, t) in enumerate(spans):
        w = state['w']['data'][e]
        if fmt == 'bf16':
            w = w.double() if case['transpose'] else w.double().T
        else:
            w = _exact_matrix(w, state['w']['sf'][e], fmt, n, k, True).T
        out[s:t] = (x[s:t] @ w) * (1.0 if state['alpha'] is None else state['alpha'][e].double())
    return out
