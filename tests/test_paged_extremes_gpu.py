"""The paged cache and its operators where values, scores and pages are extreme: rows that are left with nothing to attend
to, scores of any size, V scales and values far apart, results in memory of another layout.  Helpers and the counting of
roundings are those of test_paged_gpu."""
import math
from decimal import Context, localcontext

import pytest
import torch

from test_paged_cpu import frequencies60, two_pi
from test_paged_gpu import (BF16, DEV, E4M3, EPS, F16, F32, I8, TINY, TYPES, U, assert_turned, attention_case, check_attention, gen,
                            randn, status, values64)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype,kv', TYPES)
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('h,hkv', [(8, 2), (5, 1), (40, 2)])
@pytest.mark.parametrize('width', [40, 70, 300, 3000])
def test_sequences_without_a_page_in_the_pool_are_empty_rows(dtype, kv, d, h, hkv, width):
    """Positions whose page lies outside the pool are left out; where that is all of them the row is an empty one: zeros and
    -inf.  The widths give the batch to clusters, to the cut, and (600 positions) to pairs that lie across blocks of it."""
    from kairos_b200 import ops
    lens = [130, 600, 1, 0, 600]
    c, q, table, n = attention_case(dtype, kv, lens, h, hkv, d, 16, seed=7)
    wide = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    wide[1, :38] = -1
    wide[2, 0] = c.num_pages
    got, lse = ops.paged_attention(q, c, wide, n, return_lse=True)
    assert status() == -8
    check_attention(c, q, table, [130, 0, 0, 0, 600], got, lse)


@pytest.mark.parametrize('dtype,kv', TYPES)
def test_padded_rows_of_one_position_and_no_page(dtype, kv):
    """A captured batch's padding: length 1, a table of -1; one block a pair."""
    from kairos_b200 import ops
    c, q, table, n = attention_case(dtype, kv, [60, 1, 1], 8, 2, 128, 16)
    table[1:] = -1
    got, lse = ops.paged_attention(q, c, table, n, return_lse=True)
    assert status() == -8
    check_attention(c, q, table, [60, 0, 0], got, lse)


def level_case(dtype, kv, lens, special, width=0):
    """Keys that are 1 in channel 0 and nothing elsewhere, 2 at position special[i] of sequence i; queries 1 in channel 0."""
    c, q, table, n = attention_case(dtype, kv, lens, 8, 2, 64, 16, seed=3)
    q.zero_()
    q[..., 0] = 1
    top = {I8: 127.0, E4M3: 448.0}.get(kv, 1.0)
    row = torch.zeros(64, device=DEV)
    row[0] = top
    for i, m in enumerate(lens):
        for j in range(m):
            page, at = table[i, j // 16].item(), j % 16
            factor = 2.0 if j == special[i] else 1.0
            if c.k_scale is None:
                c.k[0, page, :, at] = (row * factor).to(kv)
            else:
                c.k[0, page, :, at].view(torch.uint8).copy_(row.to(kv).view(torch.uint8).expand(2, -1))
                c.k_scale[0, page, :, at] = factor / top
    wide = torch.full((len(lens), max(width, table.shape[1])), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    return c, q, wide, n


@pytest.mark.parametrize('dtype,kv', TYPES)
@pytest.mark.parametrize('special', [(0, 0), (3, 149), (100, 40)])
@pytest.mark.parametrize('width', [0, 2000])
def test_scores_of_any_size(dtype, kv, special, width):
    """Scores of +-2^8 to +-2^126: where one is twice the others, either it has all of the weight or the others share it
    evenly, whatever fp32 makes of them, since equal scores stay equal.  n / 16 + 64 additions, 8 U for weights and scale
    factors, 2^-16 for the weights' halves, as in check_attention."""
    from kairos_b200 import ops
    lens = [200, 150]
    c, q, table, n = level_case(dtype, kv, lens, special, width)
    v64 = c.v[0].float().double() if c.v_scale is None else c.v[0].float().double() * c.v_scale[0].double()[..., None]
    for power in (8, 20, 26, 27, 28, 29, 30, 31, 40, 100, 126):
        for sign in (1, -1):
            if power == 126 and sign == 1:
                continue                                        # the doubled score is past fp32
            got, lse = ops.paged_attention(q, c, table, n, scale=sign * 2.0 ** power, return_lse=True)
            for i, m in enumerate(lens):
                at = torch.arange(m, device=DEV)
                v = v64[table[i].long()[at // 16], :, at % 16]
                mine = at == special[i] if sign > 0 else at != special[i]
                ref, size = v[mine].mean(0), v[mine].abs().mean(0)
                tol = EPS[dtype] * ref.abs() + TINY[dtype] + size * ((m / 16 + 64) * 2 * U + 8 * U + 2.0 ** -16)
                assert ((got[i].view(2, 4, 64).double() - ref[:, None]).abs() <= tol[:, None]).all(), (power, sign, i)
                level = (2.0 if sign > 0 else -1.0) * 2.0 ** power + math.log(mine.sum().item())
                # codes: 127 * (1 / 127) and the sum of D products are off by 2 U each at the most
                assert ((lse[i].double() - level).abs() <= (m / 16 + 64) * 2 * U + 12 * U * (1 + abs(level))).all(), (power, sign, i)
    assert status() == 0


@pytest.mark.parametrize('dtype,kv', [(F16, I8), (BF16, I8), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize('h,hkv', [(8, 2), (5, 1), (40, 2)])
@pytest.mark.parametrize('ratio', [16, 24, 40, 60, 100])
@pytest.mark.parametrize('where', ['first', 'middle', 'last'])
def test_a_large_scale_of_no_weight_takes_nothing_from_the_others(dtype, kv, h, hkv, ratio, where):
    """One row of V a step of 2^ratio above the rest, its score so far below (ratio ln 2 + 20) that it adds e^-20 of the sum:
    the others keep the bits of their weights.

    Beside what check_attention counts: a head's products of weight and scale are kept times a power of two that leaves the
    largest of them, P, at 2^8 or more, as two fp16 numbers, the second of which has steps of 2^-24: half a step is 2^-33 P
    for each position, times its code.  (It shows in a channel where the row that has all of the weight has a code of 0.)"""
    from kairos_b200 import ops
    lens = [300, 70, 1000]
    c, q, table, n = attention_case(dtype, kv, lens, h, hkv, 64, 16, seed=4)
    q[..., 0] = 4
    top = {I8: 127.0, E4M3: 448.0}[kv]
    low = torch.zeros(64, device=DEV)
    low[0] = -top
    for i, m in enumerate(lens):
        j = {'first': 0, 'middle': m // 2 + 3, 'last': m - 1}[where]
        page, at = table[i, j // 16].item(), j % 16
        c.k[0, page, :, at].view(torch.uint8).copy_(low.to(kv).view(torch.uint8).expand(hkv, -1))
        c.k_scale[0, page, :, at] = (ratio * math.log(2) + 20) / (4 * top)
        c.v_scale[0, page, :, at] *= 2.0 ** ratio
    got, lse = ops.paged_attention(q, c, table, n, scale=1.0, return_lse=True)
    codes, (k64, _) = c.v[0].float().double(), values64(c)
    for i, m in enumerate(lens):
        at = torch.arange(m, device=DEV)
        pages = table[i].long()[at // 16]
        k, code, scale = (x[pages, :, at % 16].repeat_interleave(h // hkv, 1) for x in (k64, codes, c.v_scale[0].double()))
        s = torch.einsum('hd,nhd->hn', q[i].double(), k)
        p = torch.softmax(s, -1) * scale.t()                                    # products [H, n]
        ref, size = torch.einsum('hn,nhd->hd', p, code), torch.einsum('hn,nhd->hd', p, code.abs())
        ds = torch.einsum('hd,nhd->hn', q[i].double().abs(), k.abs()).amax(-1) * 72 * 2 * U
        add = (m / 16 + 64) * 2 * U
        tol = EPS[dtype] * ref.abs() + TINY[dtype] + size * (2 * ds[:, None] + add + 8 * U + 2.0 ** -16) + \
            2.0 ** -33 * p.amax(-1)[:, None] * code.abs().sum(0)
        assert ((got[i].double() - ref).abs() <= tol).all(), (i, ((got[i].double() - ref).abs() / tol).max().item())
        level = torch.logsumexp(s, -1)
        assert ((lse[i].double() - level).abs() <= ds + add + 8 * U * (1 + level.abs())).all()


@pytest.mark.parametrize('kv', [BF16, I8, E4M3])
@pytest.mark.parametrize('power', [121, 110, 60, -60, -80])
@pytest.mark.parametrize('width', [0, 2000])
def test_values_near_the_ends_of_bf16(kv, power, width):
    """Values up to 2^125 and down to 2^-80: weighted sums of them stay inside fp32."""
    from kairos_b200 import ops
    lens = [300, 1, 40, 1500]
    c, q, table, n = attention_case(BF16, kv, lens, 8, 2, 64, 16, seed=4)
    seen = torch.isfinite(c.v.float()).all(-1) if c.v_scale is None else torch.isfinite(c.v_scale)
    if c.v_scale is None:
        c.v[seen] *= 2.0 ** power
    else:
        c.v_scale[seen] *= 2.0 ** power
    wide = torch.full((4, max(width, table.shape[1])), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    got = ops.paged_attention(q, c, wide, n)
    check_attention(c, q, table, lens, got)


@pytest.mark.parametrize('h,hkv', [(8, 1), (4, 1), (16, 1)])
@pytest.mark.parametrize('gap', [10.0, 18.0, 22.0])
def test_small_weights_over_fp16_rows_beside_a_large_one(h, hkv, gap):
    """One position with all but e^-gap of the weight and values of zero: what the others add is held to 2^-37 of the largest
    weight for each of them (the halves of a weight are fp16 numbers, 2^12 at the reference, which is within 2^3 of the
    largest), beside the errors that check_attention counts."""
    from kairos_b200 import ops
    m = 5000
    c, q, table, n = attention_case(F16, F16, [m], h, hkv, 64, 16, seed=4)
    q.zero_()
    q[..., 0] = 1
    at = torch.arange(m, device=DEV)
    pages = table[0].long()[at // 16]
    c.k[0, pages, :, at % 16] = 0
    c.v[0, pages, :, at % 16] = c.v[0, pages, :, at % 16].abs() * 1024
    c.k[0, pages[7], :, 7, 0] = gap
    c.v[0, pages[7], :, 7] = 0
    got = ops.paged_attention(q, c, table, n, scale=1.0)
    v = c.v[0, pages, :, at % 16].double()
    s = torch.zeros(m, dtype=torch.float64, device=DEV)
    s[7] = gap
    p = torch.softmax(s, 0)
    ref = torch.einsum('n,nhd->hd', p, v)
    tol = EPS[F16] * ref + TINY[F16] + ref * (2 * gap * 72 * 2 * U + (m / 16 + 64) * 2 * U + 8 * U + 2.0 ** -16) + \
        2.0 ** -37 * v.sum(0) * p.max()
    assert ((got[0].view(hkv, h, 64).double() - ref[:, None]).abs() <= tol[:, None]).all()


@pytest.mark.parametrize('kv', [I8, E4M3])
@pytest.mark.parametrize('largest', [2.9e38, 3.2e38, torch.finfo(torch.bfloat16).max])
def test_queries_up_to_the_largest_bf16(kv, largest):
    """Over codes, where the queries are brought into range before the product.  (Over bf16 rows the product itself would pass
    fp32: 3e38 times a key of 2.)"""
    from kairos_b200 import ops
    lens = [200, 33]
    c, q, table, n = attention_case(BF16, kv, lens, 8, 2, 64, 16, seed=4)
    q = (q.float() * 2.0 ** 125).to(BF16)
    q[:, ::2, 5] = largest
    q[:, 1::2, 5] = -largest
    got, lse = ops.paged_attention(q, c, table, n, scale=2.0 ** -127, return_lse=True)
    check_attention(c, q, table, lens, got, lse, scale=2.0 ** -127)


def test_rotary_refuses_results_that_overlap():
    import kairos_b200 as kb
    from kairos_b200 import ops
    r, pos = kb.Rotary(64), torch.arange(5, device=DEV)
    flat = randn((5 * 40 * 64,), 1)
    x = flat.as_strided((5, 3, 64), (40 * 64, 64, 1))
    for out in (flat.as_strided((5, 3, 64), (40 * 64, 32, 1)), flat.as_strided((5, 3, 64), (64, 64, 1)),
                flat[8:].as_strided((5, 3, 64), (40 * 64, 64, 1)), flat[128:].as_strided((5, 3, 64), (40 * 64, 64, 1)),
                flat.as_strided((5, 3, 64), (40 * 64, 128, 1)), flat[576:].as_strided((5, 3, 64), (8 * 64, 64, 1))):
        kept = flat.clone()
        with pytest.raises(ValueError):
            ops.rotary(x, pos, r, out=out)
        assert torch.equal(flat, kept)
    # beside x in the same rows, in the gaps between them (320 + 512 k .. 192 further ends at 2560, where x goes on), and x itself
    # by another view
    for out in (flat[320:].as_strided((5, 3, 64), (8 * 64, 64, 1)), flat[192:].as_strided((5, 3, 64), (40 * 64, 64, 1)), flat[20 * 64:].as_strided((5, 3, 64), (40 * 64, 256, 1)), x[:]):
        kept = x.clone()
        assert ops.rotary(x, pos, r, out=out) is out
        assert_turned(out, kept, pos, r)


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
def test_rotary_into_a_result_of_other_strides(dtype):
    """x and the result have strides of their own, in 16-byte and in element-wise accesses; what lies around the result stays."""
    import kairos_b200 as kb
    from kairos_b200 import ops
    r = kb.Rotary(64, 48, layout='interleaved')
    wide = randn((4, 9, 12, 64), 1, dtype)
    odd = randn((4, 9, 12, 65), 2, dtype)
    for x in (wide[:, :, 2:9], wide.transpose(1, 2)[:, :9, :7], odd[..., 1:][:, :, 2:9], wide[:, ::1, ::2][:, :, :5]):
        b, s, h, _ = x.shape
        pos = torch.randint(0, 9999, (b, s), generator=gen(3), device=DEV)
        for room, view in ((torch.empty((s, h, b, 64), device=DEV), lambda t: t.permute(2, 0, 1, 3)),
                           (torch.empty((b, s + 2, h + 3, 64 + 16), device=DEV), lambda t: t[:, 1:-1, 2:-1, 8:72]),
                           (torch.empty((b, h, s, 64 + 3), device=DEV), lambda t: t.transpose(1, 2)[..., 1:65]),
                           (torch.empty((b * 3, s * 2, h, 64), device=DEV), lambda t: t[1::3, ::2])):
            room = torch.full_like(room, 7, dtype=dtype)
            out, kept = view(room), room.clone()
            assert ops.rotary(x, pos, r, out=out) is out
            assert_turned(out, x, pos, r)
            view(kept).copy_(out)
            assert torch.equal(room, kept)
        if b > 1:
            three = torch.full((s, 2 * h, 64), 7, dtype=dtype, device=DEV)                     # [T, H, D]
            assert_turned(ops.rotary(x[1], pos[1], r, out=three[:, 1::2]), x[1], pos[1], r)
            assert (three[:, ::2] == 7).all()


def test_rotary_of_overlapping_windows():
    """An input whose heads are windows of one row, a step of one element apart: more heads than channels, so that a result
    allocated after the input's strides would not have a dense last dimension."""
    import kairos_b200 as kb
    from kairos_b200 import ops
    r = kb.Rotary(64)
    for dtype in (F16, F32):
        flat = randn((3000,), 1, dtype)
        for shape, strides in (((2, 200, 64), (300, 1, 1)), ((3, 7, 4, 64), (1, 0, 300, 1)), ((100, 7, 1, 64), (1, 0, 300, 1))):
            x = flat.as_strided(shape, strides)
            pos = torch.randint(0, 999, shape[:-2], generator=gen(3), device=DEV)
            got = ops.rotary(x, pos, r)
            assert got.stride(-1) == 1
            assert_turned(got, x, pos, r)


@pytest.mark.parametrize('scaling', [None, dict(type='linear', factor=3.0)])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_angles_of_far_positions(scaling, layout):
    """Against angles from theta in 60 digits, not from the plan's own steps.  Beside the fp32 errors of assert_turned (8 U) the
    angle is off by 2^-32 turns for the bits that are dropped and 2^-65 turns for each position."""
    import kairos_b200 as kb
    from kairos_b200 import ops
    r = kb.Rotary(128, theta=5e5, layout=layout, scaling=scaling)
    places = [1, 1000, (1 << 24) + 1, (1 << 33) + 12345, -(1 << 33) - 7, (1 << 40) + 3, -(1 << 44)]
    pos = torch.tensor(places, device=DEV)
    x = randn((len(places), 3, 128), 1, F32)
    with localcontext(Context(prec=60)):
        steps = [f / two_pi() for f in frequencies60(128, 5e5, scaling)]
        angle = torch.tensor([[float(p * f % 1) * 2 * math.pi for f in steps] for p in places], dtype=torch.float64, device=DEV)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    i = torch.arange(64, device=DEV)
    first, second = (i, i + 64) if layout == 'half' else (2 * i, 2 * i + 1)
    a, b = x.double()[..., first], x.double()[..., second]
    got = ops.rotary(x, pos, r).double()
    tol = (a.abs() + b.abs()) * (9 * U + 2 * math.pi * (2.0 ** -32 + pos.abs().double() * 2.0 ** -65))[:, None, None]
    assert ((got[..., first] - (a * c - b * s)).abs() <= tol).all() and ((got[..., second] - (b * c + a * s)).abs() <= tol).all()
