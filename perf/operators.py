"""Cases and plain forms of the paged-cache operators: rotary positions, the rotated and quantised cache write with its
read-back, and the attention of one new token over the pages.

``run`` computes an operator in elementary torch operations (``own`` false) or through the package's entry points
(``own`` true); ``exact`` states the same definitions in 64 bits, written apart from the plain forms.
"""
import math

import torch

own = False

DTYPES = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32, 'int8': torch.int8,
          'e4m3': torch.float8_e4m3fn}
BYTES = {'f16': 2, 'bf16': 2, 'f32': 4, 'int8': 1, 'e4m3': 1}
TOP = {'int8': 127.0, 'e4m3': 448.0}          # largest magnitude of a code
THETA = 500000.0
LAYERS = 1


# ---- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small batch: q and k heads of eight tokens, launch latency
        dict(name='rotary_step', op='rotary', dtype='f16', T=8, H=40, D=128, rot=128, layout='half', scaling='none',
             factor=1.0, transpose=False, far=4096),
        # long-context prefill in bf16, most positions beyond the trained length, half of the head rotated,
        # the heads a slice of the fused projection (rows are not dense)
        dict(name='rotary_long', op='rotary', dtype='bf16', T=16381, H=32, D=128, rot=64, layout='interleaved',
             scaling='yarn', factor=4.0, transpose=False, far=131072),
        # gradient of a rotated activation kept in fp32
        dict(name='rotary_back_f32', op='rotary', dtype='f32', T=4099, H=28, D=128, rot=128, layout='half',
             scaling='llama3', factor=8.0, transpose=True, far=65536),
        # decode step of 64 sequences: one token each into an fp16 cache
        dict(name='write_step', op='write', dtype='f16', kv='f16', T=64, seqs=64, H=32, Hkv=8, D=128, rot=128,
             layout='half', scaling='llama3', factor=8.0, page=16, far=8192),
        # chunked prefill into an int8 cache; the chunk is read back for the attention that follows
        dict(name='fill_int8', op='fill', dtype='f16', kv='int8', T=4099, seqs=3, H=32, Hkv=8, D=128, rot=128,
             layout='half', scaling='none', factor=1.0, page=64, far=32768),
        # the same with an e4m3 cache, bf16 activations, a tensor-parallel shard's few heads
        dict(name='fill_e4m3', op='fill', dtype='bf16', kv='e4m3', T=16384, seqs=8, H=14, Hkv=2, D=128, rot=128,
             layout='half', scaling='yarn', factor=4.0, page=64, far=65536),
        # a cached prefix read back for a prefill that continues it
        dict(name='read_prefix', op='read', dtype='f16', kv='int8', T=50021, Hkv=8, D=128, page=64),
        # first tokens of one conversation: latency
        dict(name='attn_one_short', op='attn', dtype='f16', kv='f16', B=1, empty=0, L=300, low=300, H=32, Hkv=8, D=128,
             page=16, lse=False),
        # one long document, bf16: the cache's length has to be split
        dict(name='attn_one_long', op='attn', dtype='bf16', kv='bf16', B=1, empty=0, L=131071, low=131071, H=32, Hkv=8,
             D=128, page=64, lse=True),
        # ordinary ragged decode batch with two padded rows
        dict(name='attn_batch', op='attn', dtype='f16', kv='f16', B=32, empty=2, L=4000, low=17, H=28, Hkv=4, D=128,
             page=64, lse=True),
        # large batch over an int8 cache
        dict(name='attn_int8', op='attn', dtype='f16', kv='int8', B=128, empty=0, L=8192, low=1, H=32, Hkv=8, D=128,
             page=64, lse=False),
        # a tensor-parallel shard with one shared kv head, e4m3 cache, small pages
        dict(name='attn_e4m3', op='attn', dtype='bf16', kv='e4m3', B=24, empty=1, L=2500, low=1, H=8, Hkv=1, D=64,
             page=16, lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['rotary', 'write', 'fill', 'read', 'attn', 'attn', 'attn'])
    D = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.choice(['half', 'half', 'interleaved'])
    scaling = rng.choice(['none', 'linear', 'ntk', 'llama3', 'yarn'])
    factor = 1.0 if scaling == 'none' else rng.choice([2.0, 4.0, 8.0])
    rot = rng.choice([D, D, D // 2, D // 4])
    Hkv, G = rng.choice([(1, 8), (2, 7), (4, 7), (8, 4), (8, 8), (8, 1), (5, 3), (2, 16), (4, 12)])
    if op == 'rotary':
        D = rng.choice([64, 80, 96, 128, 256])
        H = rng.choice([1, 5, 8, 28, 32, 40])
        return dict(op=op, dtype=rng.choice(['f16', 'bf16', 'f32']), T=_log(rng, 1, 12000 * 32 * 128 // (H * D) // 4 + 2), H=H,
                    D=D, rot=rng.choice([D, D // 2]), layout=layout, scaling=scaling, factor=factor,
                    transpose=rng.choice([False, True]), far=_log(rng, 128, 200000))
    dtype = rng.choice(['f16', 'bf16'])
    kv = rng.choice([dtype, 'int8', 'e4m3'])
    if op == 'write':
        T = _log(rng, 1, 300)
        return dict(op=op, dtype=dtype, kv=dtype, T=T, seqs=T, H=Hkv * G, Hkv=Hkv, D=D, rot=rot, layout=layout,
                    scaling=scaling, factor=factor, page=16, far=_log(rng, 128, 100000))
    if op == 'fill':
        return dict(op=op, dtype=dtype, kv=kv, T=_log(rng, 2, 6000), seqs=rng.choice([1, 2, 3, 5]), H=Hkv * G, Hkv=Hkv,
                    D=D, rot=rot, layout=layout, scaling=scaling, factor=factor, page=page, far=_log(rng, 128, 100000))
    if op == 'read':
        return dict(op=op, dtype=dtype, kv=kv, T=_log(rng, 1, 50000 * 1024 // (Hkv * D) // 4 + 2), Hkv=Hkv, D=D, page=page)
    B = _log(rng, 1, 128)
    most = min(131072, 112 * 4096 * 8 * 128 // (B * Hkv * D * BYTES[kv]))
    L = _log(rng, 1, most)
    return dict(op='attn', dtype=dtype, kv=kv, B=B, empty=rng.choice([0, 0, B // 8]), L=L,
                low=rng.choice([1, max(1, L // 2), L]), H=Hkv * G, Hkv=Hkv, D=D, page=page, lse=rng.choice([False, True]))


# ---- what every form shares: lengths, scaled frequencies -----------------------------------------
def _lengths(case):
    """Ragged lengths of the batch before they are permuted; the padded rows are empty."""
    n = case['B'] - case['empty']
    low, high = case['low'], case['L']
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)] + [0] * case['empty']


def _frequencies(case):
    """Radians a position for each pair of the rotated part, and the magnitude of the rotation."""
    rot, factor, kind = case['rot'], case['factor'], case['scaling']
    i = torch.arange(rot // 2, dtype=torch.float64)
    theta = THETA * factor ** (rot / max(2, rot - 2)) if kind == 'ntk' else THETA
    f = theta ** (-2 * i / rot)
    if kind == 'linear':
        return f / factor, 1.0
    if kind == 'llama3':                       # by wavelength: trained length 8192, low and high bounds 1 and 4
        turns = 8192 * f / (2 * math.pi)       # turns within the trained length
        keep = ((turns - 1) / (4 - 1)).clamp(0, 1)
        return f * (keep + (1 - keep) / factor), 1.0
    if kind == 'yarn':                         # by pair index: trained length 32768, 32 and 1 turns
        def pair(t):
            return rot * math.log(32768 / (t * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - ramp + ramp / factor), 0.1 * math.log(factor) + 1
    return f, 1.0


def _scaling(case):
    """The same choice as the package's Rotary takes it."""
    kind = case['scaling']
    if kind == 'none':
        return None
    more = {'llama3': {'original_max': 8192}, 'yarn': {'original_max': 32768}}.get(kind, {})
    return {'type': kind, 'factor': case['factor'], **more}


# ---- inputs -------------------------------------------------------------------------------------
def _pool(case, pages, g, dev):
    """Cache pages [layer, page, head, position, D] with values as a served model leaves them, and their scales."""
    Hkv, D, page = case['Hkv'], case['D'], case['page']
    shape = (LAYERS, pages, Hkv, page, D)
    kind = case['kv']
    made = []
    for _ in range(2):
        if kind in TOP:
            scale = torch.rand(shape[:-1], generator=g, device=dev) * 0.02 + 0.01
            if kind == 'e4m3':
                scale = scale * (127.0 / 448.0)
                codes = (torch.randn(shape, generator=g, device=dev, dtype=torch.float16) * 120).clamp(-448, 448).to(DTYPES[kind])
            else:
                codes = torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8)
            made += [codes, scale]
        else:
            made += [torch.randn(shape, generator=g, device=dev, dtype=DTYPES[kind]), None]
    return dict(k=made[0], k_scale=made[1], v=made[2], v_scale=made[3])


def _slots(lens, page, g, dev):
    """Pages handed out at random to sequences of `lens` tokens: (table [B, W] int32 with -1 behind the end, pages)."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    order_host, at = order.cpu(), 0
    for b, n in enumerate(need):
        table[b, :n] = order_host[at:at + n]
        at += n
    return table.to(dev), pages


def _flat_slots(table, lens, page, dev):
    """Slot of every token, sequence after sequence."""
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(dev)
    start = torch.repeat_interleave(torch.tensor([0] + lens[:-1]).cumsum(0), torch.tensor(lens)).to(dev)
    at = torch.arange(sum(lens), device=dev) - start
    return table[seq, at // page].long() * page + at % page, at


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    op, D, dtype = case['op'], case['D'], DTYPES[case['dtype']]
    s = dict(case=case)
    if op in ('rotary', 'write', 'fill'):
        s['freq'], s['magnitude'] = _frequencies(case)
        s['freq'] = s['freq'].to(dev)
    if op == 'rotary':
        T, H = case['T'], case['H']
        # q and k heads as they lie in the fused projection: two more heads (v) behind them in every row
        s['x'] = torch.randn((T, H + 2, D), generator=g, device=dev, dtype=torch.float32).to(dtype)[:, :H]
        s['positions'] = torch.randint(0, case['far'], (T,), generator=g, device=dev)
    elif op in ('write', 'fill'):
        T, H, Hkv, n = case['T'], case['H'], case['Hkv'], min(case['seqs'], case['T'])
        s['qkv'] = torch.randn((T, (H + 2 * Hkv) * D), generator=g, device=dev, dtype=torch.float32).to(dtype)
        lens = [T // n + (i < T % n) for i in range(n)]
        table, pages = _slots(lens, case['page'], g, dev)
        s['slots'], at = _flat_slots(table, lens, case['page'], dev)
        first = torch.randint(0, case['far'], (n,), generator=g, device=dev)
        s['positions'] = at + torch.repeat_interleave(first, torch.tensor(lens, device=dev))
        if op == 'write':                      # a step: each token somewhere inside its own page
            s['slots'] = s['slots'] + torch.randint(0, case['page'], (T,), generator=g, device=dev)
        s.update(_pool(case, pages, g, dev))
    elif op == 'read':
        lens = [case['T'] - case['T'] // 3, case['T'] // 3]
        table, pages = _slots(lens, case['page'], g, dev)
        s['slots'], _ = _flat_slots(table, lens, case['page'], dev)
        s.update(_pool(case, pages, g, dev))
    else:
        lens = torch.tensor(_lengths(case))[torch.randperm(case['B'], generator=torch.Generator().manual_seed(seed))].tolist()
        s['table'], pages = _slots(lens, case['page'], g, dev)
        s['lens'] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s['q'] = torch.randn((case['B'], case['H'], D), generator=g, device=dev, dtype=torch.float32).to(dtype)
        s.update(_pool(case, pages, g, dev))
    if own:                                    # the handles that a program keeps
        import kairos_b200 as kb
        if 'freq' in s:
            s['rotary'] = kb.Rotary(D, rot_dim=case['rot'], theta=THETA, layout=case['layout'], scaling=_scaling(case),
                                    device=dev)
        if 'k' in s:
            s['cache'] = kb.PagedKVCache.from_tensors(s['k'], s['v'], s['k_scale'], s['v_scale'])
    return s


# ---- plain forms --------------------------------------------------------------------------------
def _turn(x, positions, freq, magnitude, layout, rot, back=False):
    """x [T, H, D] in fp32, the first `rot` channels rotated; angles in 64 bits (positions are far)."""
    angle = positions.double()[:, None] * freq[None, :]
    c = (torch.cos(angle) * magnitude).float()[:, None, :]
    n = (torch.sin(angle) * magnitude).float()[:, None, :]
    if back:
        n = -n
    x = x.float()
    part, rest = x[..., :rot], x[..., rot:]
    if layout == 'half':
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat((a * c - b * n, b * c + a * n), dim=-1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * c - b * n, b * c + a * n), dim=-1).flatten(-2)
    return torch.cat((part, rest), dim=-1)


def _encode(x, kind):
    """Codes and scales of rows [..., D] in fp32."""
    scale = x.abs().amax(dim=-1) / TOP[kind]
    y = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x))
    if kind == 'int8':
        return y.round().clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _put(pages, slots, page, value):
    """pages [P, Hkv, page, ...] <- value [T, Hkv, ...] at `slots`."""
    if pages.dtype == torch.float8_e4m3fn:
        pages, value = pages.view(torch.uint8), value.view(torch.uint8)
    pages[slots // page, :, slots % page] = value


def _get(pages, scales, slots, page):
    if pages.dtype == torch.float8_e4m3fn:
        got = pages.view(torch.uint8)[slots // page, :, slots % page].view(torch.float8_e4m3fn).float()
    else:
        got = pages[slots // page, :, slots % page].float()
    return got if scales is None else got * scales[slots // page, :, slots % page][..., None]


def _plain_write(s, case):
    H, Hkv, D, page = case['H'], case['Hkv'], case['D'], case['page']
    dtype = DTYPES[case['dtype']]
    x = s['qkv'].view(-1, H + 2 * Hkv, D)
    turned = _turn(x[:, :H + Hkv], s['positions'], s['freq'], s['magnitude'], case['layout'], case['rot'])
    k, v = turned[:, H:], x[:, H + Hkv:].float()
    if case['kv'] in TOP:
        (k, k_scale), (v, v_scale) = _encode(k, case['kv']), _encode(v, case['kv'])
        _put(s['k_scale'][0], s['slots'], page, k_scale)
        _put(s['v_scale'][0], s['slots'], page, v_scale)
    else:
        k, v = k.to(DTYPES[case['kv']]), v.to(DTYPES[case['kv']])
    _put(s['k'][0], s['slots'], page, k)
    _put(s['v'][0], s['slots'], page, v)
    return turned[:, :H].to(dtype)


def _plain_read(s, case):
    scales = (s['k_scale'][0], s['v_scale'][0]) if s['k_scale'] is not None else (None, None)
    return [_get(s[n][0], sc, s['slots'], case['page']).to(DTYPES[case['dtype']]) for n, sc in zip('kv', scales)]


def _plain_attention(s, case):
    q, lens, table = s['q'], s['lens'].long(), s['table'].long().clamp(min=0)
    B, H, D = q.shape
    Hkv = case['Hkv']
    got = []
    for pages, scale in ((s['k'][0], s['k_scale']), (s['v'][0], s['v_scale'])):
        x = (pages.view(torch.uint8)[table].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[table]).float()
        if scale is not None:
            x = x * scale[0][table][..., None]
        got.append(x.transpose(1, 2).reshape(B, Hkv, -1, D))            # [B, Hkv, W * page, D]
    k, v = got
    seen = torch.arange(k.shape[2], device=q.device)[None, :] < lens[:, None]
    v = torch.where(seen[:, None, :, None], v, torch.zeros_like(v))
    score = torch.matmul(q.view(B, Hkv, H // Hkv, D).float(), k.transpose(2, 3)) * (1 / math.sqrt(D))
    score = torch.where(seen[:, None, None, :], score, torch.full_like(score, float('-inf')))
    top = score.amax(dim=-1, keepdim=True)
    some = (lens > 0)[:, None, None, None]
    weight = torch.where(some, torch.exp(score - torch.where(some, top, torch.zeros_like(top))), torch.zeros_like(score))
    total = weight.sum(dim=-1, keepdim=True)
    out = torch.matmul(weight, v) / torch.where(some, total, torch.ones_like(total))
    lse = torch.where(some, top + torch.log(total), torch.full_like(total, float('-inf')))
    out = out.reshape(B, H, D).to(q.dtype)
    return (out, lse.reshape(B, H)) if case['lse'] else out


def run(state):
    s, case = state, state['case']
    op = case['op']
    if own:
        from kairos_b200 import ops
        if op == 'rotary':
            return ops.rotary(s['x'], s['positions'], s['rotary'], transpose=case['transpose'])
        if op == 'write':
            return [ops.rope_paged_kv(s['qkv'], s['positions'], s['slots'], s['rotary'], s['cache']), s['k'], s['v']]
        if op == 'fill':
            q = ops.rope_paged_kv(s['qkv'], s['positions'], s['slots'], s['rotary'], s['cache'])
            return [q, *ops.paged_kv_read(s['cache'], s['slots'], dtype=q.dtype)]
        if op == 'read':
            return list(ops.paged_kv_read(s['cache'], s['slots'], dtype=DTYPES[case['dtype']]))
        return ops.paged_attention(s['q'], s['cache'], s['table'], s['lens'], return_lse=case['lse'])
    if op == 'rotary':
        return _turn(s['x'], s['positions'], s['freq'], s['magnitude'], case['layout'], case['rot'],
                     case['transpose']).to(s['x'].dtype)
    if op == 'write':
        return [_plain_write(s, case), s['k'], s['v']]
    if op == 'fill':
        return [_plain_write(s, case), *_plain_read(s, case)]
    if op == 'read':
        return _plain_read(s, case)
    return _plain_attention(s, case)


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    op, D, e = case['op'], case['D'], BYTES[case['dtype']]
    c = BYTES.get(case.get('kv'), 0)
    scale = 4 if case.get('kv') in TOP else 0
    if op == 'rotary':
        return {'bytes': case['T'] * (2 * case['H'] * D * e + 8), 'flops': case['T'] * case['H'] * case['rot'] * 3}
    if op in ('write', 'fill'):
        T, H, Hkv = case['T'], case['H'], case['Hkv']
        bytes_ = T * ((2 * H + 2 * Hkv) * D * e + 2 * Hkv * (D * c + scale) + 16)
        if op == 'fill':                       # and read back
            bytes_ += T * (2 * Hkv * (D * c + scale + D * e) + 8)
        return {'bytes': bytes_, 'flops': T * ((H + Hkv) * case['rot'] * 3 + (2 * Hkv * D * 3 if scale else 0))}
    if op == 'read':
        T, Hkv = case['T'], case['Hkv']
        return {'bytes': T * (2 * Hkv * (D * c + scale + D * e) + 8), 'flops': T * 2 * Hkv * D}
    tokens, B, H, Hkv = sum(_lengths(case)), case['B'], case['H'], case['Hkv']
    return {'bytes': tokens * 2 * Hkv * (D * c + scale) + 2 * B * H * D * e + -(-tokens // case['page']) * 4 + B * 4,
            'flops': 4 * tokens * H * D}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _exact_frequency(case, i):
    rot, factor, kind = case['rot'], case['factor'], case['scaling']
    if kind == 'ntk':                          # the base grows so that the slowest pair is slowed by `factor`
        return 1.0 / math.pow(THETA * math.pow(factor, rot / max(2, rot - 2)), 2 * i / rot)
    f = 1.0 / math.pow(THETA, 2 * i / rot)
    if kind == 'linear':
        return f / factor
    if kind == 'llama3':
        wavelength = 2 * math.pi / f
        if wavelength < 8192 / 4:
            return f
        if wavelength > 8192 / 1:
            return f / factor
        part = (8192 / wavelength - 1) / 3
        return (1 - part) * f / factor + part * f
    if kind == 'yarn':
        first = max(0, math.floor(rot / 2 * math.log(32768 / (2 * math.pi * 32)) / math.log(THETA)))
        last = min(rot - 1, math.ceil(rot / 2 * math.log(32768 / (2 * math.pi)) / math.log(THETA)))
        part = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
        return part * f / factor + (1 - part) * f
    return f


def _exact_turn(x, positions, case, back=False):
    """Pairs as complex numbers, multiplied by magnitude * exp(+-i * position * frequency)."""
    rot = case['rot']
    freq = torch.tensor([_exact_frequency(case, i) for i in range(rot // 2)], dtype=torch.float64)
    magnitude = 1 + 0.1 * math.log(case['factor']) if case['scaling'] == 'yarn' else 1.0
    unit = torch.polar(torch.full((), magnitude, dtype=torch.float64, device=x.device).expand(x.shape[0], rot // 2).contiguous(),
                       torch.outer(positions.double(), freq.to(x.device)) * (-1 if back else 1))[:, None]
    y = x.double().clone()
    if case['layout'] == 'half':
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * unit
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.complex(y[..., 0:rot:2].contiguous(), y[..., 1:rot:2].contiguous()) * unit
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def _exact_held(x, kind):
    """The value that a quantised row stands for."""
    if kind not in TOP:
        return x
    scale = x.abs().amax(dim=-1, keepdim=True) / TOP[kind]
    y = x / scale
    if kind == 'int8':
        return torch.round(y) * scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)    # e4m3: three bits behind the first
    return torch.round(y / step) * step * scale


def _value(s, name, page, offset):
    x = s[name][0][page, :, offset] if s[name].dtype != torch.float8_e4m3fn else \
        s[name][0].view(torch.uint8)[page, :, offset].view(torch.float8_e4m3fn)
    x = x.double()
    return x if s[name + '_scale'] is None else x * s[name + '_scale'][0][page, :, offset].double()[..., None]


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case['op']
    if op == 'rotary':
        return _exact_turn(s['x'], s['positions'], case, case['transpose'])
    if op in ('write', 'fill'):
        H, Hkv, D, page = case['H'], case['Hkv'], case['D'], case['page']
        heads = s['qkv'].view(-1, H + 2 * Hkv, D)
        q, k = _exact_turn(heads[:, :H], s['positions'], case), _exact_turn(heads[:, H:H + Hkv], s['positions'], case)
        k, v = _exact_held(k, case['kv']), _exact_held(heads[:, H + Hkv:].double(), case['kv'])
        if op == 'fill':
            return [q, k, v]
        whole = []
        for name, new in (('k', k), ('v', v)):
            full = s[name].double()
            full[0, s['slots'] // page, :, s['slots'] % page] = new
            whole.append(full)
        return [q, *whole]
    page = case['page']
    if op == 'read':
        return [_value(s, n, s['slots'] // page, s['slots'] % page) for n in 'kv']
    B, H, D = s['q'].shape
    out = torch.zeros((B, H, D), dtype=torch.float64, device=s['q'].device)
    lse = torch.full((B, H), float('-inf'), dtype=torch.float64, device=s['q'].device)
    for b, n in enumerate(s['lens'].tolist()):
        if n:
            at = torch.arange(n, device=out.device)
            pages = s['table'][b].long()[at // page]
            k, v = _value(s, 'k', pages, at % page), _value(s, 'v', pages, at % page)       # [n, Hkv, D]
            score = torch.einsum('hgd,nhd->hgn', s['q'][b].double().view(case['Hkv'], -1, D), k) / math.sqrt(D)
            out[b] = torch.einsum('hgn,nhd->hgd', torch.softmax(score, dim=-1), v).reshape(H, D)
            lse[b] = torch.logsumexp(score, dim=-1).reshape(H)
    return (out, lse) if case['lse'] else out
