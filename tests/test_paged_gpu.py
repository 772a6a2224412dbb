"""Rotary positions, the paged cache's write and read-back, and the attention of one new token over the pages, against
plain 64-bit statements.

Tolerances count roundings.  U = 2^-24 is half a step of fp32; EPS[t] half a step of the output type, relative to the value
(finfo.eps / 2), beside the half step of its subnormals."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
F16, BF16, F32, I8, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn
YARN = dict(type='yarn', factor=4.0, original_max=32768)
LLAMA3 = dict(type='llama3', factor=8.0, original_max=8192)
DEV = 'cuda'


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(shape, seed, dtype=F16):
    return torch.randn(shape, generator=gen(seed), device=DEV, dtype=F32).to(dtype)


def status():
    from kairos_b200 import runtime
    torch.cuda.synchronize()
    return runtime.device_status(clear=True)


# ---- rotary ------------------------------------------------------------------------------------------
def turn64(x, positions, r, back=False):
    """The rotation in 64 bits, and the sum |a| + |b| of every pair (what fp32 errors are relative to)."""
    rot = r.rot_dim
    # the angle modulo a turn as an exact integer product: 64-bit floats lose 1e-16 * position radians
    turns = (positions[..., None] * r.steps).double() * 2.0 ** -64
    c, s = torch.cos(turns * 2 * math.pi)[..., None, :] * r.magnitude, torch.sin(turns * 2 * math.pi)[..., None, :] * r.magnitude
    s = -s if back else s
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    i = torch.arange(rot // 2, device=x.device)
    first, second = (i, i + rot // 2) if r.layout == 'half' else (2 * i, 2 * i + 1)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * r.magnitude
    return y, size


def assert_turned(got, x, positions, r, back=False):
    """fp32 errors of a turned value, in U * (|a| + |b|) * magnitude: the angle as fp32 half turns (2^-25 * pi: 1.6), sin and cos
    (2), times the magnitude (1), two products and a sum (2): under 8.  Then one rounding to the output type."""
    ref, size = turn64(x, positions, r, back)
    tol = EPS[got.dtype] * ref.abs() + (1 + EPS[got.dtype]) * 8 * U * size + TINY[got.dtype]
    assert ((got.double() - ref).abs() <= tol).all()
    assert torch.equal(got[..., r.rot_dim:], x[..., r.rot_dim:])


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('d,rot,scaling', [(128, 128, None), (128, 32, YARN), (64, 64, LLAMA3), (80, 40, None), (96, 96, dict(type='ntk', factor=2.)),
                                           (256, 64, dict(type='linear', factor=3.)), (33, 20, None), (2, 2, None), (512, 512, YARN)])
def test_rotary(dtype, layout, d, rot, scaling):
    import kairos_b200 as kb
    from kairos_b200 import ops
    r = kb.Rotary(d, rot, theta=5e5, layout=layout, scaling=scaling)
    for t, h in ((1, 1), (3, 5), (70, 28), (257, 2)):
        x = randn((t, h, d), t * 7 + h, dtype)
        pos = torch.randint(-10, 1 << 20, (t,), generator=gen(t), device=DEV)
        pos[0] = 0
        pos[-1] = (1 << 33) + 12345                            # far: the 64-bit product has to wrap
        assert_turned(ops.rotary(x, pos, r), x, pos, r)
        assert_turned(ops.rotary(x, pos, r, transpose=True), x, pos, r, back=True)


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
def test_rotary_strides_shapes_and_in_place(dtype):
    import kairos_b200 as kb
    from kairos_b200 import ops
    r = kb.Rotary(64, 48, layout='half')
    wide = randn((4, 9, 12, 64), 1, dtype)
    views = [wide[:, :, 2:9], wide.transpose(1, 2)[:, 1:5], wide[1:2, ::3], wide.transpose(0, 1), wide[:, 4], wide[:, :1, :1],
             randn((4, 9, 7, 68), 2, dtype)[..., 2:66], randn((4, 9, 7, 65), 3, dtype)[..., 1:]]      # the last two: odd alignment
    for x in views:
        pos = torch.randint(0, 9999, x.shape[:-2], generator=gen(3), device=DEV)
        assert_turned(ops.rotary(x, pos, r), x, pos, r)
        kept = x.clone()
        out = torch.zeros_like(wide) if x.shape == wide.shape else None
        assert ops.rotary(x, pos, r, out=x) is x
        assert_turned(x, kept, pos, r)
        del out
    x = randn((3, 5, 2, 64), 4, dtype)
    row = torch.arange(5, device=DEV)                           # one row of positions for the whole batch
    assert_turned(ops.rotary(x, row, r), x, row.expand(3, 5), r)
    col = torch.arange(3, device=DEV)[:, None]
    assert_turned(ops.rotary(x, col, r), x, col.expand(3, 5), r)
    assert_turned(ops.rotary(x, torch.arange(10, device=DEV)[::2], r), x, (2 * row).expand(3, 5), r)
    assert ops.rotary(x[:0], row, r).shape == (0, 5, 2, 64) and ops.rotary(x[:, :, :0], row, r).numel() == 0


def test_rotary_refuses_on_device():
    import kairos_b200 as kb
    from kairos_b200 import ops
    r, x, pos = kb.Rotary(64), randn((3, 2, 64), 1), torch.arange(3, device=DEV)
    for call in (lambda: ops.rotary(x, pos.int(), r), lambda: ops.rotary(x, pos.cpu(), r), lambda: ops.rotary(x, pos, r, out=x.float()),
                 lambda: ops.rotary(x, pos, r, out=x[:2]), lambda: ops.rotary(x, pos, kb.Rotary(64, device='cpu'))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        ops.rotary(x, torch.arange(4, device=DEV), r)


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_rotary_transpose_is_the_gradient(layout):
    """<R x, g> against <x, R^T g>, and R^T g against central differences of <R x, g> -- exact for a linear operator but for
    the roundings, which are bounded as in assert_turned: per element 8 U (|a| + |b|) m + U |y|."""
    import kairos_b200 as kb
    from kairos_b200 import ops
    r = kb.Rotary(64, 32, layout=layout, scaling=YARN)
    x, g = randn((5, 3, 64), 1, F32), randn((5, 3, 64), 2, F32)
    pos = torch.randint(0, 50000, (5,), generator=gen(3), device=DEV)
    back = ops.rotary(g, pos, r, transpose=True)
    assert_turned(back, g, pos, r, back=True)
    _, size = turn64(x, pos, r)
    _, gsize = turn64(g, pos, r)
    slack = (8 * U * size + U * (size + x.abs())) * g.abs() + (8 * U * gsize + U * (gsize + g.abs())) * x.abs()
    assert abs((ops.rotary(x, pos, r).double() * g).sum() - (x.double() * back).sum()) <= slack.sum()
    for at in ((0, 0, 0), (2, 1, 17), (4, 2, 31), (1, 0, 40)):
        h = 0.5
        up, down = x.clone(), x.clone()
        up[at] += h
        down[at] -= h
        step = (up[at].double() - down[at].double()).item()
        diff = ((ops.rotary(up, pos, r).double() - ops.rotary(down, pos, r).double()) * g).sum().item() / step
        # only the pair of `at` differs: two elements, each rounded on both sides
        err = 2 * 2 * (10 * U * (x[at[:2]].abs().max().item() + 1) * 2 * r.magnitude * g[at[:2]].abs().max().item()) / step
        assert abs(diff - back[at].item()) <= err + 10 * U * gsize[at].item()


# ---- cache write and read-back --------------------------------------------------------------------------
def held64(x, kv):
    """What a cached row stands for, and how far a stored value may be from x: half a step of its code."""
    if kv in (F16, BF16):
        return EPS[kv] * x.abs() + TINY[kv]
    top = {I8: 127.0, E4M3: 448.0}[kv]
    amax = x.abs().amax(-1, keepdim=True)
    if kv is I8:
        return amax / top / 2 * (1 + 1e-5) + 0 * x
    return torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * amax / top) * (1 + 1e-5)


def make_cache(kv, heads, d, page=16, pages=12, seed=0, layers=2):
    """A cache whose every byte is known beforehand (codes and scales of some earlier use)."""
    import kairos_b200 as kb
    c = kb.PagedKVCache(layers, pages, heads, d, page, kv)
    for t in (c.k, c.v):
        t.view(torch.uint8).copy_(torch.randint(0, 100, t.view(torch.uint8).shape, generator=gen(seed), device=DEV).to(torch.uint8))
    for s in (c.k_scale, c.v_scale):
        if s is not None:
            s.copy_(torch.rand(s.shape, generator=gen(seed + 1), device=DEV))
    return c


def raw(c, layer=None):
    ts = [t if t.dtype is F32 else t.view(torch.uint8) for t in (c.k, c.v, c.k_scale, c.v_scale) if t is not None]
    return [t.clone() if layer is None else t[layer].clone() for t in ts]


@pytest.mark.parametrize('dtype,kv', [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('d,rot,h,hkv,page', [(128, 128, 32, 8, 64), (64, 64, 4, 1, 16), (128, 64, 7, 1, 32), (256, 64, 3, 3, 128), (64, 16, 28, 4, 256)])
def test_write_and_read(dtype, kv, layout, d, rot, h, hkv, page):
    import kairos_b200 as kb
    from kairos_b200 import ops
    r = kb.Rotary(d, rot, theta=5e5, layout=layout, scaling=YARN)
    for t in (1, 2, 37, 130):
        c = make_cache(kv, hkv, d, page, pages=-(-3 * t // page) + 2)
        before = raw(c)
        qkv = randn((t, (h + 2 * hkv) * d + 16), t, dtype)[:, 8:-8]                  # strided rows
        pos = torch.randint(0, 200000, (t,), generator=gen(t), device=DEV)
        slots = torch.randperm(c.num_pages * page, generator=gen(5), device=DEV)[:t].contiguous()
        if t > 2:
            slots[1] = -1                                                             # padding
        q = ops.rope_paged_kv(qkv, pos, slots, r, c, layer=1)
        x = qkv.reshape(t, h + 2 * hkv, d)
        assert_turned(q, x[:, :h], pos, r)
        real = slots >= 0
        k64, size = turn64(x[:, h:h + hkv], pos, r)
        for name, ref, fp32 in (('k', k64, 8 * U * size), ('v', x[:, h + hkv:].double(), 0 * size)):
            # the row's largest value carries its own fp32 error into every value of the row by way of the scale
            slack = fp32 + fp32.amax(-1, keepdim=True) if kv in (I8, E4M3) else fp32
            for out in (F32, dtype):
                got = dict(zip('kv', ops.paged_kv_read(c, slots, layer=1, dtype=out)))[name]
                tol = held64(ref, kv) + 2 * slack
                tol = tol + (EPS[out] + 2 * U) * (ref.abs() + tol) + TINY[out]
                assert ((got.double() - ref).abs() <= tol)[real].all()
                assert (got[~real] == 0).all()
        # everything else of the pool, of the other layer too, is as it was
        live = slots[real]
        for was, now in zip(before, raw(c)):
            now[1, live // page, :, live % page] = was[1, live // page, :, live % page]
            assert torch.equal(was, now)


@pytest.mark.parametrize('kv', [I8, E4M3])
def test_quantised_rows_are_the_nearest_codes(kv):
    """V is not turned, so its codes follow from fp32 arithmetic alone: equal to torch's, value for value."""
    import kairos_b200 as kb
    from kairos_b200 import ops
    t, d, top = 300, 128, {I8: 127.0, E4M3: 448.0}[kv]
    x = randn((t, 3, d), 3)
    x[0] = 0
    x[1, 2] = 6e-8                                              # the smallest fp16: scales far below fp16's range
    x[2, 2, 5] = 65504.
    x[3, 2] = torch.arange(d, device=DEV).half() - 64           # ties at the quotient's half steps
    x[4, 2] = 0.5
    c, slots = make_cache(kv, 1, d, 16, 20), torch.arange(t, device=DEV)
    ops.rope_paged_kv(x.view(t, -1), slots, slots, kb.Rotary(d), c)
    v = x[:, 2].float()
    scale = v.abs().amax(-1) / torch.full((t,), top, device=DEV)
    y = torch.where(scale[:, None] > 0, v / scale[:, None], torch.zeros_like(v))
    code = y.round().clamp(-127, 127).to(I8) if kv is I8 else y.clamp(-448, 448).to(E4M3)
    got, gs = c.v[0].transpose(1, 2).reshape(-1, d)[:t], c.v_scale[0].transpose(1, 2).reshape(-1)[:t]
    assert torch.equal(gs, scale) and torch.equal(got.float(), code.float())
    assert (ops.paged_kv_read(c, slots)[0][0] == 0).all()       # a row of zeros reads back as zeros


@pytest.mark.parametrize('kv', [I8, E4M3])
def test_rows_that_are_not_finite_read_back_as_nan(kv):
    import kairos_b200 as kb
    from kairos_b200 import ops
    x = randn((6, 3, 64), 3)
    x[1, 1, 7], x[2, 2, 0], x[3, 2, 63], x[4, 1, 5] = float('nan'), float('inf'), float('-inf'), float('inf')
    c, slots = make_cache(kv, 1, 64), torch.arange(6, device=DEV)
    ops.rope_paged_kv(x.view(6, -1), slots, slots, kb.Rotary(64), c)
    k, v = ops.paged_kv_read(c, slots)
    for rows, bad in ((k, (1, 4)), (v, (2, 3))):
        for i in range(6):
            assert torch.isnan(rows[i]).all() if i in bad else torch.isfinite(rows[i]).all()


def test_slots_past_the_pool_are_refused_on_the_device():
    import kairos_b200 as kb
    from kairos_b200 import ops
    c, r = make_cache(F16, 2, 64, 16, 4), kb.Rotary(64)
    x, pos = randn((3, 8 * 64), 1), torch.arange(3, device=DEV)
    assert status() == 0
    before = raw(c)
    q = ops.rope_paged_kv(x, pos, torch.tensor([64, 3, 1 << 40], device=DEV), r, c)
    assert status() == -8 and status() == 0
    assert_turned(q, x.view(3, 8, 64)[:, :4], pos, r)
    for was, now in zip(before, raw(c)):
        now[0, 0, :, 3] = was[0, 0, :, 3]
        assert torch.equal(was, now)
    k, v = ops.paged_kv_read(c, torch.tensor([3, 64], device=DEV))
    assert status() == -8 and (k[1] == 0).all() and (v[1] == 0).all()
    assert torch.equal(v[0], x.view(3, 8, 64)[1, 6:])


def test_write_and_read_refuse_on_device():
    import kairos_b200 as kb
    from kairos_b200 import ops
    c, r = make_cache(F16, 2, 64), kb.Rotary(64)
    x, pos = randn((3, 8 * 64), 1), torch.arange(3, device=DEV)
    for call in (lambda: ops.rope_paged_kv(x.bfloat16(), pos, pos, r, c), lambda: ops.rope_paged_kv(x, pos, pos, kb.Rotary(64, 20), c)):
        with pytest.raises(kb.KairosError):
            call()
    for call in (lambda: ops.rope_paged_kv(x, pos.int(), pos, r, c), lambda: ops.rope_paged_kv(x, pos, pos[:2], r, c),
                 lambda: ops.rope_paged_kv(x, pos, pos.cpu(), r, c), lambda: ops.rope_paged_kv(x, pos, pos, r, c, q_out=x),
                 lambda: ops.rope_paged_kv(x, torch.arange(6, device=DEV)[::2], pos, r, c),
                 lambda: ops.paged_kv_read(c, pos.int()), lambda: ops.paged_kv_read(c, pos, out=(x, x))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(IndexError):
        ops.paged_kv_read(c, pos, layer=2)
    assert ops.rope_paged_kv(x[:0], pos[:0], pos[:0], r, c).shape == (0, 4, 64)
    assert ops.paged_kv_read(c, pos[:0])[0].shape == (0, 2, 64)


# ---- attention -------------------------------------------------------------------------------------------
def fill(c, seed=0, layer=0, spread=1.0):
    """Cached values as a served model leaves them, in every position of the pool."""
    for i, (t, s) in enumerate(((c.k, c.k_scale), (c.v, c.v_scale))):
        if s is None:
            t[layer].copy_(randn(t.shape[1:], seed + i, c.kv_dtype) * spread)
            continue
        top = 127 if c.kv_dtype is I8 else 448
        x = torch.rand(t.shape[1:], generator=gen(seed + i), device=DEV) * 2 * top - top
        if c.kv_dtype is I8:
            t[layer].copy_(x.round().to(I8))
        else:
            t[layer].view(torch.uint8).copy_(x.to(E4M3).view(torch.uint8))
        s[layer].copy_((torch.rand(s.shape[1:], generator=gen(seed + 2 + i), device=DEV) + 0.5) / top * spread * 2)


def values64(c, layer=0):
    out = []
    for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = t[layer].float().double()
        out.append(x if s is None else x * s[layer].double()[..., None])
    return out


def check_attention(c, q, table, lens, got, lse=None, layer=0, scale=None):
    """Against 64 bits.  With D channels and n keys: a score is a sum of D products, off by (D + 8) U sum |q k| * scale (the
    tensor unit may cut instead of round: 2 U), a weight by that and 4 U of the exponential and its scale factors; weights
    and values are added n / 16 times at the least coarse and joined in 64 more steps; one rounding at the end.  Weights
    enter the second product as two 16-bit halves: 2^-16 of each at the most."""
    k64, v64 = values64(c, layer)
    b, h, d = q.shape
    group, page = h // c.kv_heads, c.page_size
    scale = d ** -0.5 if scale is None else scale
    for i, n in enumerate(lens):
        if n <= 0:
            assert (got[i] == 0).all() and (lse is None or (lse[i] == -math.inf).all())
            continue
        at = torch.arange(n, device=DEV)
        pages = table[i].long()[at // page]
        k, v = (x[pages, :, at % page].repeat_interleave(group, 1) for x in (k64, v64))       # [n, H, D]
        s = torch.einsum('hd,nhd->hn', q[i].double(), k) * scale
        p = torch.softmax(s, -1)
        ref = torch.einsum('hn,nhd->hd', p, v)
        ds = (torch.einsum('hd,nhd->hn', q[i].double().abs(), k.abs()) * abs(scale)).amax(-1) * (d + 8) * 2 * U
        add = (n / 16 + 64) * 2 * U
        weigh = torch.einsum('hn,nhd->hd', p, v.abs())
        tol = EPS[q.dtype] * ref.abs() + TINY[q.dtype] + weigh * (2 * ds[:, None] + add + 8 * U + 2.0 ** -16)
        assert ((got[i].double() - ref).abs() <= tol).all(), (i, n, ((got[i].double() - ref).abs() / tol).max().item())
        if lse is not None:
            ref = torch.logsumexp(s, -1)
            assert ((lse[i].double() - ref).abs() <= ds + add + 8 * U * (1 + ref.abs())).all()


def attention_case(dtype, kv, lens, h, hkv, d, page, seed=0, spare=2):
    """Cache, table with random pages (and -1 behind each end) and queries; every position that no length covers holds NaN,
    infinities, or (codes) NaN scales."""
    import kairos_b200 as kb
    need = [-(-max(0, n) // page) for n in lens]
    c = kb.PagedKVCache(1, sum(need) + spare, hkv, d, page, kv)
    fill(c, seed)
    order = torch.randperm(c.num_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need, default=0) + 1), -1, dtype=torch.int32)
    unused = torch.ones(c.num_pages, page, dtype=torch.bool)
    for i, n in enumerate(need):
        mine, order = order[:n], order[n:]
        table[i, :n] = torch.tensor(mine, dtype=torch.int32)
        for j, pg in enumerate(mine):
            unused[pg, :max(0, min(page, lens[i] - j * page))] = False
    unused = unused.to(DEV)[None, :, None, :].expand(1, -1, hkv, -1)
    for x, s, bad in ((c.k, c.k_scale, float('nan')), (c.v, c.v_scale, float('inf'))):
        if s is not None:
            s[unused] = float('nan')
            x.view(torch.uint8)[unused] = 0x7f                  # e4m3: NaN
        else:
            x[unused] = bad
    q = randn((len(lens), h, d), seed + 9, dtype)
    return c, q, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


TYPES = [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8), (F16, E4M3), (BF16, E4M3)]
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 257, 500, 1023, 0]


@pytest.mark.parametrize('dtype,kv', TYPES)
@pytest.mark.parametrize('d,page', [(64, 16), (128, 16), (128, 64), (256, 32), (64, 256)])
@pytest.mark.parametrize('h,hkv', [(8, 1), (4, 4), (28, 4), (9, 3), (16, 1), (12, 1), (40, 2)])
def test_attention(dtype, kv, d, page, h, hkv):
    from kairos_b200 import ops
    c, q, table, lens = attention_case(dtype, kv, LENGTHS, h, hkv, d, page, seed=h + d)
    got, lse = ops.paged_attention(q, c, table, lens, return_lse=True)
    check_attention(c, q, table, LENGTHS, got, lse)
    assert status() == 0


@pytest.mark.parametrize('dtype,kv', TYPES)
@pytest.mark.parametrize('lens,h,hkv,d', [([40001], 8, 1, 128), ([1], 4, 4, 64), ([30000, 3, 0, 9000], 28, 4, 128), ([4097], 64, 8, 256),
                                          ([100] * 300, 16, 8, 64), ([0, 0], 4, 2, 128), ([0], 1, 1, 128), ([700, 1] * 20, 32, 8, 128)])
def test_attention_long_and_many(dtype, kv, lens, h, hkv, d):
    from kairos_b200 import ops
    c, q, table, n = attention_case(dtype, kv, lens, h, hkv, d, 64, seed=5)
    got, lse = ops.paged_attention(q, c, table, n, return_lse=True)
    check_attention(c, q, table, lens, got, lse)
    again, lse2 = ops.paged_attention(q, c, table, n, return_lse=True)
    assert torch.equal(got, again) and torch.equal(lse, lse2)          # no order of arrival in the result


@pytest.mark.parametrize('dtype,kv', TYPES)
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('lens', [[1], [64], [65, 0, 3], [600], [129, 1025], [1023, 0, 511, 513, 1, 900], [4000, 17], [257] * 40,
                                  [2500, 1, 0, 64, 640] * 5])
@pytest.mark.parametrize('h,hkv', [(5, 1), (24, 2)])
def test_attention_whatever_shares_the_work(dtype, kv, d, lens, h, hkv):
    """The table's width decides whether blocks, clusters of 2, 4 or 8 blocks, or a cut by the lengths on the device share a
    sequence: the same lengths with tables of growing width, every result against 64 bits."""
    from kairos_b200 import ops
    c, q, table, n = attention_case(dtype, kv, lens, h, hkv, d, 16, seed=len(lens) + d)
    ref = None
    for width in (table.shape[1], 70, 140, 300, 900, 3000):
        if width < table.shape[1]:
            continue
        wide = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        got, lse = ops.paged_attention(q, c, wide, n, return_lse=True)
        if ref is None or not torch.equal(got, ref[0]) or not torch.equal(lse, ref[1]):
            check_attention(c, q, table, lens, got, lse)
            ref = got, lse
    assert status() == 0


@pytest.mark.parametrize('dtype,kv', TYPES)
def test_attention_peaked_scores_and_scale(dtype, kv):
    """Scores tens apart, so that running maxima keep changing; a scale of its own, zero and negative ones."""
    from kairos_b200 import ops
    lens = [2000, 333, 64]
    c, q, table, n = attention_case(dtype, kv, lens, 8, 2, 128, 32, seed=2)
    for scale in (1.0, 0.0, -0.7, 3.0):
        got, lse = ops.paged_attention(q, c, table, n, scale=scale, return_lse=True)
        check_attention(c, q, table, lens, got, lse, scale=scale)


@pytest.mark.parametrize('kv', [I8, E4M3])
@pytest.mark.parametrize('dtype', [F16, BF16])
def test_attention_scales_of_very_different_size(dtype, kv):
    """Rows of V whose scales span forty binary orders: each keeps its own share of the sum."""
    from kairos_b200 import ops
    lens = [300, 70]
    c, q, table, n = attention_case(dtype, kv, lens, 8, 2, 64, 16, seed=4)
    c.v_scale *= torch.exp2(torch.randint(-30, 11, c.v_scale.shape, generator=gen(1), device=DEV).float())
    q = q * 3
    got = ops.paged_attention(q, c, table, n)
    check_attention(c, q, table, lens, got)
    one = [1, 0]                                                # a single row with a tiny scale
    c.v_scale[torch.isfinite(c.v_scale)] = 2.0 ** -12
    check_attention(c, q, table, one, ops.paged_attention(q, c, table, torch.tensor(one, dtype=torch.int32, device=DEV)))


@pytest.mark.parametrize('scale_q', [2.0 ** -60, 2.0 ** 60, 0.0])
def test_attention_bf16_queries_beyond_fp16(scale_q):
    """bf16 queries over coded caches keep their range: 2^+-60 with the inverse in the softmax's scale."""
    from kairos_b200 import ops
    for kv in (I8, E4M3):
        c, q, table, n = attention_case(BF16, kv, [200], 8, 2, 64, 16, seed=4)
        q = q * scale_q
        s = 0.1 / scale_q if scale_q else 1.0
        got, lse = ops.paged_attention(q, c, table, n, scale=s, return_lse=True)
        check_attention(c, q, table, [200], got, lse, scale=s)


def test_attention_strides_tables_and_out():
    from kairos_b200 import ops
    lens = [70, 0, 130]
    c, q, table, n = attention_case(F16, F16, lens, 8, 2, 64, 16)
    ref = ops.paged_attention(q, c, table, n)
    wide = torch.zeros((3, 12, 72), dtype=F16, device=DEV)
    wide[:, 2:10, 8:] = q
    assert torch.equal(ops.paged_attention(wide[:, 2:10, 8:], c, table, n), ref)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.paged_attention(turned, c, table, n), ref)
    wide_table = torch.full((3, table.shape[1] + 5), 1 << 30, dtype=torch.int32, device=DEV)
    wide_table[:, :table.shape[1]] = table
    assert torch.equal(ops.paged_attention(q, c, wide_table, n), ref)
    assert torch.equal(ops.paged_attention(q, c, wide_table[:, :table.shape[1]], n), ref)
    out = torch.full_like(ref, 7)
    assert ops.paged_attention(q, c, table, n, out=out) is out and torch.equal(out, ref)
    own = q.clone()
    assert ops.paged_attention(own, c, table, n, out=own) is own and torch.equal(own, ref)     # the result over the queries
    # one sequence's pages shared by the whole batch (stride 0)
    many = ops.paged_attention(q[2:].expand(4, -1, -1).contiguous(), c, table[2:].expand(4, -1), n[2:].expand(4).contiguous())
    assert all(torch.equal(m, ref[2]) for m in many)
    assert ops.paged_attention(q[:0], c, table[:0], n[:0]).shape == (0, 8, 64)
    assert (ops.paged_attention(q, c, table[:, :0], torch.zeros_like(n)) == 0).all()
    assert (ops.paged_attention(q, c, table, torch.full_like(n, -5)) == 0).all()
    assert status() == 0


def test_attention_bad_pages_and_lengths_are_reported():
    from kairos_b200 import ops
    lens = [70, 40, 130]
    c, q, table, n = attention_case(F16, F16, lens, 8, 2, 64, 16)
    ref = ops.paged_attention(q, c, table, n)
    bad = table.clone()
    bad[1, 1], bad[1, 0] = 1 << 30, -7
    got = ops.paged_attention(q, c, bad, n)
    assert status() == -8
    assert torch.equal(got[0], ref[0]) and torch.equal(got[2], ref[2])
    bad = table[:, :4].contiguous()                             # shorter than 70 and 130
    got = ops.paged_attention(q, c, bad, n)
    assert status() == -8
    check_attention(c, q, table, [64, 40, 64], got)
    c2, q2, table2, n2 = attention_case(F16, F16, [64, 1], 4, 1, 64, 16)
    table2[0, 2] = c2.num_pages                                 # one of four pages: its 16 positions are left out
    kept = [0, 1, 3]
    got = ops.paged_attention(q2, c2, table2, n2)
    assert status() == -8
    short = table2.clone()
    short[0, :3] = table2[0, kept]
    check_attention(c2, q2, short, [48, 1], got)


@pytest.mark.parametrize('kv', [F16, I8])
def test_attention_values_that_are_not_finite(kv):
    """A NaN among the seen positions makes its head's row NaN (as the formula does), and no other."""
    from kairos_b200 import ops
    lens = [100, 100]
    c, q, table, n = attention_case(F16, kv, lens, 8, 2, 64, 16)
    ref = ops.paged_attention(q, c, table, n)
    (c.k if kv is F16 else c.k_scale)[0, table[0, 3], 1, 5] = float('nan')
    got = ops.paged_attention(q, c, table, n)
    assert torch.isnan(got[0, 4:]).all() and torch.equal(got[0, :4], ref[0, :4]) and torch.equal(got[1], ref[1])
    if kv is F16:
        c, q, table, n = attention_case(F16, kv, lens, 8, 2, 64, 16)
        q[0, 0, 3], q[0, 0, 4:] = 1.0, 0.0
        q[0, 0, :3] = 0
        c.k[0, table[0, 2], 0, 7, 3] = float('-inf')            # one score of -inf: that position has weight zero
        got = ops.paged_attention(q, c, table, n)
        c.k[0, table[0, 2], 0, 7, 3] = -30000.0
        low = ops.paged_attention(q, c, table, n)
        assert torch.equal(got[0, 0], low[0, 0])
        c.k[0, table[0, 2], 0, 7, 3] = float('inf')             # of +inf: inf - inf
        assert torch.isnan(ops.paged_attention(q, c, table, n)[0, 0]).all()


def test_attention_refuses_on_device():
    import kairos_b200 as kb
    from kairos_b200 import ops
    c, q, table, n = attention_case(F16, F16, [20, 30], 8, 2, 64, 16)
    for call in (lambda: ops.paged_attention(q[:, :3], c, table, n), lambda: ops.paged_attention(q.bfloat16(), c, table, n),
                 lambda: ops.paged_attention(randn((2, 8, 68), 1)[..., 2:66], c, table, n)):
        with pytest.raises(kb.KairosError):
            call()
    for call in (lambda: ops.paged_attention(q, c, table.long(), n), lambda: ops.paged_attention(q, c, table[:1], n),
                 lambda: ops.paged_attention(q, c, table, n.long()), lambda: ops.paged_attention(q, c, table, n[:1]),
                 lambda: ops.paged_attention(q, c, table.t().contiguous().t(), n), lambda: ops.paged_attention(q, c, table, n, out=q[:1]),
                 lambda: ops.paged_attention(q, c, table.cpu(), n), lambda: ops.paged_attention(q, c, table, n, out=q.float())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(IndexError):
        ops.paged_attention(q, c, table, n, layer=1)


def test_attention_far_into_a_large_pool():
    """Row offsets past 2^31 elements: only the last pages of a pool of 4.3 G elements are used."""
    import kairos_b200 as kb
    from kairos_b200 import ops
    pages = (1 << 31) // (8 * 64 * 128) + 40
    c = kb.PagedKVCache(1, pages, 8, 128, 64, I8)
    lens = [150, 200]
    table = torch.tensor([[pages - 1, pages - 3, pages - 2, -1], [pages - 9, 0, pages - 7, pages - 5]], dtype=torch.int32, device=DEV)
    total = sum(lens)
    slots = torch.cat([table[i].long()[torch.arange(n, device=DEV) // 64] * 64 + torch.arange(n, device=DEV) % 64 for i, n in enumerate(lens)])
    qkv = randn((total, 24 * 128), 1)
    ops.rope_paged_kv(qkv, torch.arange(total, device=DEV), slots, kb.Rotary(128), c)
    k, v = ops.paged_kv_read(c, slots, dtype=F32)
    q = randn((2, 8, 128), 2)
    got = ops.paged_attention(q, c, table, torch.tensor(lens, dtype=torch.int32, device=DEV))
    first = 0
    for i, n in enumerate(lens):
        s = torch.einsum('hd,nhd->hn', q[i].double(), k[first:first + n].double()) * 128 ** -0.5
        ref = torch.einsum('hn,nhd->hd', torch.softmax(s, -1), v[first:first + n].double())
        assert (got[i].double() - ref).abs().max() <= 2.0 ** -11 * ref.abs().max() + 1e-4      # scores: 136 * 2 U * 3 sqrt(128) / 11 ~ 5e-5, twice
        first += n
    assert status() == 0


# ---- streams, graphs, and the operators together ------------------------------------------------------------
def test_other_streams_and_graphs_side_by_side():
    """Two captured graphs of the same shapes replayed at once on two streams (workspaces of their own), with lengths that
    change between replays; an eager call on a third stream meanwhile."""
    from kairos_b200 import ops
    lens = [3000, 17, 800, 0]
    c, q, table, n = attention_case(F16, F16, lens, 32, 4, 128, 64)
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    torch.cuda.synchronize()
    for i in range(2):
        qi, ni = (q * (1 - 2 * i)).clone(), n.clone()
        with torch.cuda.stream(streams[i]):
            ops.paged_attention(qi, c, table, ni)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            out = ops.paged_attention(qi, c, table, ni)
        graphs.append((g, qi, ni, out))
    for shift in (0, 5, 900):
        now = [max(0, m - shift) for m in lens]
        for _, _, ni, _ in graphs:
            ni.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(20):
            for i, (g, *_rest) in enumerate(graphs):
                with torch.cuda.stream(streams[i]):
                    g.replay()
            with torch.cuda.stream(streams[2]):
                eager = ops.paged_attention(q, c, table, graphs[0][2])
        torch.cuda.synchronize()
        for _, qi, _, out in graphs:
            check_attention(c, qi, table, now, out)
        assert torch.equal(eager, graphs[0][3])
    assert status() == 0


@pytest.mark.parametrize('dtype,kv', TYPES)
def test_operators_together(dtype, kv):
    """Prefill of ragged prompts, then decode steps captured into one graph, as a serving loop runs them: the cache's pages
    grow and the result equals attention over everything written, as the cache holds it."""
    import kairos_b200 as kb
    from kairos_b200 import ops
    h, hkv, d, page, prompts, steps = 8, 2, 64, 16, [37, 0, 5], 20
    c = kb.PagedKVCache(1, 16, hkv, d, page, kv)
    r = kb.Rotary(d, 32, layout='interleaved', scaling=YARN)
    for i, n in enumerate(prompts):
        c.reserve(i, n + steps)
    slots, positions = c.slots(range(3), prompts)
    ops.rope_paged_kv(randn((sum(prompts), (h + 2 * hkv) * d), 1, dtype), positions, slots, r, c)
    table = c.page_table(range(3))
    lens = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    qkv = randn((3, (h + 2 * hkv) * d), 0, dtype)

    def step():
        at = lens.long()
        slot = table.gather(1, (at // page)[:, None])[:, 0].long() * page + at % page
        q = ops.rope_paged_kv(qkv, at, slot, r, c)
        lens.add_(1)
        return q, ops.paged_attention(q, c, table, lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    lens.copy_(torch.tensor(prompts, dtype=torch.int32))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        q, out = step()
    lens.copy_(torch.tensor(prompts, dtype=torch.int32))
    for i in range(steps):
        qkv.copy_(randn(qkv.shape, 10 + i, dtype))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check_attention(c, q, table, [n + i + 1 for n in prompts], out)
    # the pages hold what was written: the last token's row of every sequence
    at = lens.long() - 1
    slot = table.gather(1, (at // page)[:, None])[:, 0].long() * page + at % page
    _, v = ops.paged_kv_read(c, slot, dtype=F32)
    x = qkv.view(3, -1, d)[:, h + hkv:].double()
    assert ((v.double() - x).abs() <= held64(x, kv) * (1 + 1e-5) + 1e-12).all()
    assert status() == 0


def test_rotary_refuses_a_result_that_overlaps_itself():
    import kairos_b200 as kb
    from kairos_b200 import ops
    r, one, pos = kb.Rotary(64), randn((1, 2, 64), 1), torch.arange(3, device=DEV)
    x = one.expand(3, 2, 64)                                    # broadcast inputs are fine, broadcast results are not
    assert_turned(ops.rotary(x, pos, r), x, pos, r)
    with pytest.raises(ValueError):
        ops.rotary(x, pos, r, out=x)
    with pytest.raises(ValueError):
        ops.rotary(x, pos, r, out=torch.empty((3, 1, 64), dtype=F16, device=DEV).expand(3, 2, 64))
    assert ops.rotary(one, pos[:1], r, out=torch.empty_like(one).expand(1, 2, 64)).shape == one.shape
