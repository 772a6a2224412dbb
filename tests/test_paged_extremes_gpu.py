"""The paged cache and its operators where values, scores and pages are extreme: rows that are left with nothing to attend
to, scores of any size, V scales and values far apart, results in memory of another layout.  Helpers and the counting of
roundings are those of test_paged_gpu."""
import math

import pytest
import torch

from test_paged_gpu import (BF16, DEV, E4M3, EPS, F16, F32, I8, TINY, TYPES, U, assert_turned, attention_case, check_attention, gen,
                            randn, status)

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
