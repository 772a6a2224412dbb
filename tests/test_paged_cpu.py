"""Paged cache and rotary positions, the parts without a GPU: page accounting, frequencies, and every refusal -- of the
operators' argument checks and of the C entry points (which refuse before anything is launched)."""
import ctypes
import math
from decimal import Context, Decimal, localcontext

import pytest
import torch

import kairos_b200 as kb
from kairos_b200 import _lib, ops

lib = _lib.lib
SHAPE, ALIGN, ARG = -1, -2, -8


def cache(**kw):
    args = dict(layers=2, num_pages=6, kv_heads=2, head_dim=64, page_size=16, kv_dtype='float16', device='cpu')
    args.update(kw)
    return kb.PagedKVCache(**args)


# ---- page accounting -----------------------------------------------------------------------------
def test_pages_are_handed_out_and_taken_back():
    c = cache()
    assert c.reserve('a', 17) == c.reserve('a', 3) and len(c.reserve('a', 32)) == 2
    c.reserve('b', 0)
    c.reserve('b', 49)
    assert c.free_pages == 0
    with pytest.raises(kb.KairosError):
        c.reserve('a', 33)
    assert len(c.reserve('a', 32)) == 2                      # the refused call changed nothing
    table = c.page_table(['b', 'a'])
    assert table.dtype == torch.int32 and table.shape == (2, 4) and table[1, 2:].tolist() == [-1, -1]
    used = [p for p in table.flatten().tolist() if p >= 0]
    assert sorted(used) == list(range(6))
    with pytest.raises(ValueError):
        c.page_table(['b'], width=3)
    assert c.page_table(['a'], width=5).shape == (1, 5) and c.page_table([]).shape == (0, 0)
    c.release('b')
    assert c.free_pages == 4
    with pytest.raises(KeyError):
        c.release('b')
    with pytest.raises(ValueError):
        c.reserve('a', -1)


def test_slots_follow_the_pages():
    c = cache()
    c.reserve('x', 20)
    c.reserve('y', 5)
    slots, positions = c.slots(['x', 'y'], [18, 5], [2, 0])
    pages = c.page_table(['x', 'y'])
    assert positions.tolist() == list(range(2, 20)) + list(range(5))
    assert slots.tolist() == [int(pages[0, p // 16]) * 16 + p % 16 for p in range(2, 20)] + [int(pages[1, 0]) * 16 + p for p in range(5)]
    for bad in (([33], [0]), ([1], [-1]), ([16], [17])):
        with pytest.raises(ValueError):
            c.slots(['x'], *bad)
    assert c.slots([], [])[0].numel() == 0


def test_cache_refusals():
    for kw in (dict(kv_dtype='int4'), dict(page_size=24), dict(head_dim=96), dict(num_pages=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            cache(**kw)
    k = torch.zeros(1, 2, 1, 16, 64, dtype=torch.int8)
    s = torch.zeros(1, 2, 1, 16)
    kb.PagedKVCache.from_tensors(k, k.clone(), s, s.clone())
    t, ts = torch.zeros(1, 16, 1, 16, 64, dtype=torch.int8).transpose(1, 3), torch.zeros(1, 16, 1, 16)
    for args in ((k, k, None, None), (k, k, s, s.half()), (k, k.half(), s, s), (k, k, s, s[:, :1]), (k.half(), k.half(), s, s),
                 (k[0], k[0], s, s), (t, t, ts, ts)):
        with pytest.raises(ValueError):
            kb.PagedKVCache.from_tensors(*args)


# ---- frequencies ---------------------------------------------------------------------------------
def test_steps_are_binary_fractions_of_a_turn():
    r = kb.Rotary(128, theta=10000.0, device='cpu')
    for i, step in enumerate(r.steps.tolist()):
        f = 10000.0 ** (-2 * i / 128)
        assert abs((step % (1 << 64)) / 2.0 ** 64 - f / (2 * math.pi)) <= 2e-16 * f + 2.0 ** -64
    far = 10_000_019
    turns = (far * r.steps[0].item()) % (1 << 64) / 2.0 ** 64
    assert abs(math.cos(2 * math.pi * turns) - math.cos(far)) < 1e-8      # the fp64 angle itself is good to 1e-9


@pytest.mark.parametrize('scaling', [None, dict(type='linear', factor=4), dict(type='ntk', factor=4),
                                     dict(type='llama3', factor=8, original_max=8192),
                                     dict(type='yarn', factor=4, original_max=32768)])
def test_scaled_frequencies(scaling):
    base, r = kb.Rotary(128, 64, theta=5e5, device='cpu'), kb.Rotary(128, 64, theta=5e5, scaling=scaling, device='cpu')
    ratio = r.frequencies / base.frequencies
    factor = scaling['factor'] if scaling else 1
    assert ((ratio >= 1 / factor - 1e-12) & (ratio <= 1 + 1e-12)).all() and abs(ratio[-1] - 1 / factor) < 1e-9
    assert (ratio[1:] <= ratio[:-1] + 1e-12).all()
    if scaling and scaling['type'] not in ('linear',):
        assert abs(ratio[0] - 1) < 1e-12                      # the fastest pair keeps its speed
    assert r.magnitude == pytest.approx(0.1 * math.log(4) + 1 if scaling and scaling['type'] == 'yarn' else 1.0)


@pytest.mark.parametrize('kw', [dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=130), dict(layout='both'), dict(theta=1.0),
                                dict(scaling={'type': 'linear'}), dict(scaling={'type': 'other', 'factor': 2}),
                                dict(scaling={'type': 'linear', 'factor': 0.5}), dict(scaling={'type': 'llama3', 'factor': 2}),
                                dict(scaling={'type': 'linear', 'factor': 2, 'more': 1}),
                                dict(scaling={'type': 'llama3', 'factor': 2, 'original_max': 10, 'low_freq_factor': 4})])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        kb.Rotary(128, device='cpu', **kw)


# ---- operators: everything that is not on one CUDA device or of a wrong form ------------------------
def test_operators_refuse_cpu_tensors_and_wrong_forms():
    c, r = cache(), kb.Rotary(64, device='cpu')
    x, pos = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int64)
    slots, table, lens = pos, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.float16)
    for call in (lambda: ops.rotary(x, pos, r), lambda: ops.rope_paged_kv(qkv, pos, slots, r, c),
                 lambda: ops.paged_kv_read(c, slots), lambda: ops.paged_attention(x, c, table, lens)):
        with pytest.raises(ValueError, match='CUDA'):
            call()
    for call in (lambda: ops.rotary(x.double(), pos, r), lambda: ops.rotary(x[0], pos, r), lambda: ops.rotary(x[..., :32], pos, r),
                 lambda: ops.rotary(x.transpose(1, 2), pos, r),
                 lambda: ops.rope_paged_kv(qkv.float(), pos, slots, r, c), lambda: ops.rope_paged_kv(qkv[:, :256], pos, slots, r, c),
                 lambda: ops.rope_paged_kv(qkv[:, :-1], pos, slots, r, c), lambda: ops.rope_paged_kv(qkv, pos, slots, kb.Rotary(128, device='cpu'), c),
                 lambda: ops.paged_kv_read(c, slots, dtype=torch.int8), lambda: ops.paged_attention(x.float(), c, table, lens),
                 lambda: ops.paged_attention(x[..., :32], c, table, lens), lambda: ops.paged_attention(x[0], c, table, lens)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(IndexError):
        c.layer_ptrs[2]


# ---- C entry points: refused before a launch ---------------------------------------------------------
P = 0x1000            # aligned addresses that are never touched: every call below is refused


def layer(**kw):
    args = dict(k=P, v=P, k_scale=None, v_scale=None, pages=4, kv_heads=2, page_size=16, head_dim=64, dtype=0)
    args.update(kw)
    return _lib.KvLayer(**args)


BAD_LAYERS = [(dict(pages=0), SHAPE), (dict(kv_heads=-1), SHAPE), (dict(page_size=8), SHAPE), (dict(page_size=48), SHAPE),
              (dict(page_size=512), SHAPE), (dict(head_dim=96), SHAPE), (dict(k=None), ALIGN), (dict(v=P + 8), ALIGN),
              (dict(dtype=2), ARG), (dict(dtype=3), ALIGN), (dict(dtype=4, k_scale=P), ALIGN)]


def attention(kv, q=P, strides=(256, 64), table=P, table_stride=4, width=4, lens=P, o=P, lse=None, b=2, h=4, dtype=0, ws=P, wsb=1 << 30):
    return lib.kairos_paged_attention(q, *strides, ctypes.addressof(kv), table, table_stride, width, lens, o, lse, b, h, 1.0,
                                      dtype, ws, wsb, None)


def write(kv, qkv=P, stride=512, pos=P, slots=P, plan=(P, 1.0, 64, 0), q=P, t=3, h=4, dtype=0):
    pl = _lib.RotaryPlan(*plan)
    return lib.kairos_rope_paged_kv(qkv, stride, pos, slots, ctypes.addressof(pl), ctypes.addressof(kv), q, t, h, dtype, None)


def turn(x=P, y=P, pos=P, plan=(P, 1.0, 64, 0), dtype=0, b=1, s=3, h=4, d=64):
    pl = _lib.RotaryPlan(*plan)
    return lib.kairos_rotary(x, 0, 256, 64, y, 0, 256, 64, pos, 0, 1, ctypes.addressof(pl), dtype, 0, b, s, h, d, None)


@pytest.mark.parametrize('kw,code', BAD_LAYERS)
def test_c_refuses_bad_pools(kw, code):
    kv = layer(**kw)
    assert attention(kv) == code and write(kv) == code
    assert lib.kairos_paged_kv_read(ctypes.addressof(kv), P, P, P, 3, 0, None) == code


@pytest.mark.parametrize('kw,code', [(dict(b=-1), SHAPE), (dict(h=3), SHAPE), (dict(h=0), SHAPE), (dict(width=-1), SHAPE),
                                     (dict(b=65536), SHAPE), (dict(width=1 << 28), SHAPE), (dict(dtype=1), ARG), (dict(dtype=2), ARG),
                                     (dict(q=None), ALIGN), (dict(q=P + 2), ALIGN), (dict(strides=(256, 63)), ALIGN),
                                     (dict(o=P + 8), ALIGN), (dict(lens=None), ALIGN), (dict(lse=P + 2), ALIGN), (dict(table=None), ALIGN),
                                     (dict(table_stride=-1), SHAPE)])
def test_c_refuses_attention(kw, code):
    assert attention(layer(), **kw) == code


@pytest.mark.parametrize('kw,code', [(dict(t=-1), SHAPE), (dict(h=0), SHAPE), (dict(stride=511), SHAPE), (dict(stride=504), SHAPE),
                                     (dict(plan=(P, 1.0, 24, 0)), ARG), (dict(plan=(P, 1.0, 80, 0)), ARG), (dict(plan=(None, 1.0, 64, 0)), ARG),
                                     (dict(plan=(P, 1.0, 64, 2)), ARG), (dict(dtype=1), ARG), (dict(dtype=2), ARG), (dict(q=P + 4), ALIGN),
                                     (dict(qkv=None), ALIGN), (dict(slots=P + 4), ALIGN), (dict(pos=None), ALIGN)])
def test_c_refuses_write(kw, code):
    assert write(layer(), **kw) == code


@pytest.mark.parametrize('kw,code', [(dict(d=0), SHAPE), (dict(d=513), SHAPE), (dict(s=-1), SHAPE), (dict(b=1 << 17, s=1 << 17), SHAPE),
                                     (dict(plan=(P, 1.0, 66, 0)), ARG), (dict(plan=(P, 1.0, 31, 0)), ARG), (dict(dtype=3), ARG),
                                     (dict(x=None), ALIGN), (dict(pos=P + 4), ALIGN)])
def test_c_refuses_rotary(kw, code):
    assert turn(**kw) == code


def test_empty_calls_need_no_device():
    assert attention(layer(), b=0) == 0 and write(layer(), t=0) == 0 and turn(s=0) == 0 and turn(h=0) == 0
    assert lib.kairos_paged_kv_read(ctypes.addressof(layer()), P, P, P, 0, 0, None) == 0


def test_pages_of_a_sequence_are_a_copy():
    c = cache()
    assert c.pages('a') == []
    c.reserve('a', 17)
    held = c.pages('a')
    assert held == c.page_table(['a'])[0].tolist() and len(held) == 2
    held.append(5)
    assert len(c.pages('a')) == 2 and c.free_pages == 4


# ---- results that would overlap ----------------------------------------------------------------------
LAYOUTS = [((3, 2, 4), (8, 4, 1)), ((3, 2, 4), (0, 4, 1)), ((3, 2, 4), (8, 2, 1)), ((3, 2, 4), (4, 12, 1)), ((3, 2, 4), (4, 4, 1)),
           ((2, 3, 4), (12, 4, 1)), ((2, 3, 4), (6, 4, 1)), ((3, 2, 2), (4, 6, 1)), ((3, 2, 2), (3, 2, 1)), ((1, 2, 4), (0, 4, 1)),
           ((2, 3, 2, 4), (40, 8, 4, 1)), ((2, 3, 2, 4), (24, 4, 12, 1)), ((2, 3, 2, 4), (4, 8, 24, 1)), ((0, 2, 4), (0, 0, 1)),
           ((2, 2, 1), (2, 1, 1)), ((2, 2, 1), (1, 1, 1))]


def elements(shape, strides, offset=0):
    at = [offset]
    for n, step in zip(shape, strides):
        at = [a + i * step for a in at for i in range(n)]
    return at


@pytest.mark.parametrize('shape,strides', LAYOUTS)
def test_results_whose_elements_share_a_place(shape, strides):
    at = elements(shape, strides)
    assert ops._distinct(shape, strides) == (len(set(at)) == len(at))


@pytest.mark.parametrize('shape,strides', [x for x in LAYOUTS if 0 not in x[0]])
def test_results_that_overlap_their_input(shape, strides):
    for s, other in LAYOUTS:
        if s != shape:
            continue
        first = set(elements(shape, strides))
        for offset in range(-70, 71):
            assert ops._disjoint(shape, strides, other, offset) == first.isdisjoint(elements(shape, other, offset)), (other, offset)


# ---- the kernels' steps against the definition in 60 digits -----------------------------------------------
def two_pi():
    def arctan_inverse(x):                                    # of 1 / x, by its series
        total, term, n = Decimal(0), 1 / Decimal(x), 0
        while abs(term) > Decimal('1e-70'):
            total += term / (2 * n + 1) * (-1) ** n
            term, n = term / (x * x), n + 1
        return total
    return 8 * (4 * arctan_inverse(5) - arctan_inverse(239))  # Machin


def frequencies60(rot, theta, scaling):
    """Radians a position, from the definitions of the scalings."""
    kind, s = (scaling or {}).get('type'), Decimal((scaling or {}).get('factor', 1))
    theta = Decimal(theta)
    if kind == 'ntk':
        theta = theta * s ** (Decimal(rot) / max(2, rot - 2))
    out = []
    for i in range(rot // 2):
        f = theta ** (Decimal(-2 * i) / rot)
        if kind == 'linear':
            f = f / s
        elif kind == 'llama3':                                # trained 8192, low 1, high 4
            wavelength = two_pi() / f
            part = (Decimal(8192) / wavelength - 1) / 3
            f = f if wavelength < 2048 else f / s if wavelength > 8192 else (1 - part) * f / s + part * f
        elif kind == 'yarn':                                  # trained 32768, 32 and 1 turns
            at = [Decimal(rot) / 2 * (32768 / (two_pi() * t)).ln() / theta.ln() for t in (32, 1)]
            first, last = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
            part = min(Decimal(1), max(Decimal(0), (Decimal(i) - first) / (last - first)))
            f = part * f / s + (1 - part) * f
        out.append(f)
    return out


@pytest.mark.parametrize('rot', [2, 20, 64, 128])
@pytest.mark.parametrize('theta', [10000.0, 5e5, 1234567.891])
@pytest.mark.parametrize('scaling', [None, dict(type='linear', factor=3), dict(type='ntk', factor=4), dict(type='llama3', factor=8, original_max=8192),
                                     dict(type='yarn', factor=2.5, original_max=32768)])
def test_steps_are_rounded_once(rot, theta, scaling):
    """Half a step of 2^-64 turns, so that a far position multiplies nothing else; the frequencies half a step of fp64."""
    with localcontext(Context(prec=60)):
        r = kb.Rotary(128, rot, theta=theta, scaling=scaling, device='cpu')
        for step, kept, f in zip(r.steps.tolist(), r.frequencies.tolist(), frequencies60(rot, theta, scaling)):
            off = (step - f / two_pi() * (1 << 64)) % (1 << 64)
            assert min(off, (1 << 64) - off) <= Decimal('0.5000001')
            assert abs(Decimal(kept) - f) <= f * Decimal(2) ** -53


def test_slices_of_one_activation_are_told_apart_at_once(monkeypatch):
    """The usual neighbours -- heads of another kind in the same rows, batched or not -- without a look at every row."""
    monkeypatch.setattr(ops, '_rows', None)
    row, heads = 40 * 64, 8
    for shape, strides in (((4096, heads, 64), (row, 64, 1)), ((32, 4096, heads, 64), (4096 * row, row, 64, 1)),
                           ((heads, 4096, 64), (64, row, 1)), ((1, 4096, heads, 64), (7, row, 64, 1))):
        assert ops._distinct(shape, strides)
        for offset in (heads * 64, -heads * 64, 20 * 64, 4096 * row * 40):
            assert ops._disjoint(shape, strides, strides, offset)
