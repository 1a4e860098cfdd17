"""A long chunk among many sequences of one token: by the rows that a sequence brings on average the call takes tiles of few rows, and
the chunk is many of them."""
import pytest
import torch

import svod_amd
from svod_amd import Attn
import pages_reference as ref
from pages_reference import draw_lengths, make
from test_gpu_pages_places import KINDS, held, normal

pytestmark = pytest.mark.gpu


def step(device, batch, chunk, at, h, hkv, d, page, dtype, coded, context=400, long=0, rows_after=0):
    """`batch` sequences that bring a token each, the `at`-th of them `chunk`; `long`: earlier tokens of one more than most have."""
    contexts, _ = draw_lengths(batch + d, batch, context, 1)
    if long:
        contexts[batch // 2] = long
    fresh = [chunk if b == at else 1 for b in range(batch)]
    return make(device, contexts, fresh, kv_heads=hkv, d=d, page=page, dtype=dtype, coded=coded, seed=batch, rows_after=rows_after)


def both(device, case, h, opts, splits=None):
    q = normal((case.rows, h, case.k.shape[3]), case.dtype, 3, device)
    got = svod_amd.attention_paged(q, case.pages, Attn(splits=splits, **opts))
    form = svod_amd.chosen()
    held(got, *ref.attention(case, q, **opts), form)
    again = svod_amd.attention_paged(q, case.pages, Attn(splits=splits, **opts))
    sequences = slice(case.starts[0], case.starts[-1])
    assert torch.equal(got[sequences].view(torch.int16), again[sequences].view(torch.int16))
    return form


@pytest.mark.parametrize("dtype,coded", KINDS)
@pytest.mark.parametrize("opts", [dict(causal=True), dict(causal=True, window=(20, 0)), dict(causal=True, window=(300, 0)), {}])
@pytest.mark.parametrize("batch,chunk,at,h,hkv,d,rows", [
    (64, 449, 30, 4, 1, 64, 32),     # 57 tiles of 8 tokens
    (64, 449, 0, 4, 1, 128, 32),
    (64, 961, 63, 4, 2, 64, 32),     # 61 tiles of 16 tokens
    (70, 500, 69, 2, 2, 64, 16),     # 32 tiles of 16
    (70, 200, 5, 4, 1, 128, 16),
    (70, 170, 33, 4, 2, 256, 16)])
def test_a_long_chunk_among_single_tokens(device, batch, chunk, at, h, hkv, d, rows, opts, dtype, coded):
    case = step(device, batch, chunk, at, h, hkv, d, 16, dtype, coded)
    assert f"rows: {rows}," in both(device, case, h, opts)


@pytest.mark.parametrize("dtype,coded", KINDS)
@pytest.mark.parametrize("splits", [None, 3])
@pytest.mark.parametrize("batch,chunk,h,hkv,d,rows", [(64, 449, 32, 8, 128, 32), (100, 700, 8, 8, 64, 16)])
def test_a_long_chunk_in_shares_and_parts(device, batch, chunk, h, hkv, d, rows, splits, dtype, coded):
    """Contexts long enough that keys are split: shares that take many tiles of the chunk, and a long sequence beside it."""
    case = step(device, batch, chunk, 3, h, hkv, d, 16, dtype, coded, context=1500, long=9000)
    q = torch.empty(case.rows, h, d, dtype=dtype, device=device)
    assert svod_amd.attention_paged_workspace(q, case.pages, Attn(causal=True, splits=splits)) > 0
    assert f"rows: {rows}," in both(device, case, h, dict(causal=True), splits)


@pytest.mark.parametrize("dtype,coded", KINDS)
def test_the_same_chunk_in_the_other_form(device, dtype, coded):
    """Rows of no sequence count with the others: with a few the same step takes tiles of 128 rows."""
    for rows_after, rows in ((0, 32), (8, 128)):
        case = step(device, 64, 449, 10, 4, 1, 64, 32, dtype, coded, rows_after=rows_after)
        assert f"rows: {rows}," in both(device, case, 4, dict(causal=True))
