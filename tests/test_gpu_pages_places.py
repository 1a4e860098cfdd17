"""Rows of a step that have no place in a cache in pages, or none that is there: what write_pages stores and attention_paged sees."""
import pytest
import torch

import svod_amd
from svod_amd import Attn, Pages
import pages_reference as ref
from pages_reference import make

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
KINDS = [(BF16, False), (F16, False), (BF16, True), (F16, True)]


def bits(x):
    return x.detach().cpu().contiguous().view(torch.uint8 if x.element_size() == 1 else torch.int16)


def normal(shape, dtype, seed, device, by=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * by).to(dtype).to(device)


def held(got, want, allowed, what=""):
    got, rows = got.double().cpu(), ~torch.isnan(want)
    assert torch.isfinite(got[rows]).all(), what
    off = (got - want).abs()[rows]
    assert not (off > allowed[rows]).any(), (what, float((off - allowed[rows]).max()))


# ---- write_pages: a row goes to its own position, or nowhere.
def stored(table, lens, starts, rows, columns, page, count):
    """(row, page, row of the page) of each packed row that has a place: the definition, on whole numbers of any size."""
    for b in range(len(lens)):
        for row in range(max(starts[b], 0), min(starts[b + 1], rows)):
            at = lens[b] - (starts[b + 1] - row)
            if 0 <= at < columns * page and 0 <= table[b][at // page] < count:
                yield row, table[b][at // page], at % page


@pytest.mark.parametrize("dtype,coded", KINDS)
@pytest.mark.parametrize("name", ["pages that are none", "no page at all", "lengths past the table", "lengths far out", "ends past the rows"])
@pytest.mark.parametrize("hkv,new", [(2, [5, 3, 40, 1]), (8, [900, 1, 800, 350])])
@pytest.mark.parametrize("wide", [torch.int64, torch.int32])
def test_a_row_goes_to_its_place_or_nowhere(device, wide, hkv, new, name, dtype, coded):
    """Entries, lengths and starts out of range, beside sequences that are as they should be: nothing is written to a page or a
    position that is not the row's own.  (The larger call takes four heads a wave.)"""
    d, page = 128, 16
    case = make(device, [37, 0, 70, 16], new, kv_heads=hkv, d=d, page=page, dtype=dtype, coded=coded, seed=hkv, fill=0.0, rows_after=3,
                wide=(wide, wide))
    lens, starts, table, rows, count = list(case.lens), list(case.starts), case.table.clone(), case.rows, case.k.shape[0]
    columns = table.shape[1]
    if name == "pages that are none":
        table[0, -(-lens[0] // page) - 1] = -1
        table[2, lens[2] // page // 2 + 2] = count
        table[3, (lens[3] - 1) // page] = 0x7fffffff
    elif name == "no page at all":
        table[0] = -1
        table[2] = -(1 << 31)
        table[3] = count
    elif name == "lengths past the table":
        lens[0] = columns * page + 2
        lens[2] = columns * page + new[2] - 1
        lens[3] = columns * page + new[3]
    elif name == "lengths far out":
        far = torch.iinfo(wide)
        lens[0], lens[2], lens[3] = far.max, far.min, (1 << 32) + 5 if wide == torch.int64 else far.max // 2
    else:
        starts[4] = rows + 2  # two rows more than there are
    # A place named twice would be a wrong test.
    places = list(stored(table.tolist(), lens, starts, rows, columns, page, count))
    assert len({(i, r) for _, i, r in places}) == len(places)
    k, v = (normal((rows, hkv, d), dtype, s, "cpu", by=3.0) for s in (1, 2))
    pages = Pages(case.pages.k, case.pages.v, table.to(device), torch.tensor(lens, dtype=wide, device=device),
                  torch.tensor(starts, dtype=wide, device=device), case.pages.scales)
    pools = [case.pages.k, case.pages.v, *(case.pages.scales or ())]
    want = [bits(x).clone() for x in pools]
    # The same rows by a call that has nothing out of range: one sequence of them all.
    clean = make(device, [0], [rows], kv_heads=hkv, d=d, page=page, dtype=dtype, coded=coded, seed=0, fill=0.0)
    svod_amd.write_pages(k.to(device), v.to(device), clean.pages)
    own = [bits(x) for x in (clean.pages.k, clean.pages.v, *(clean.pages.scales or ()))]
    for row, i, r in places:
        for to, x in zip(want, own):
            to[i, :, r] = x[int(clean.table[0, row // page]), :, row % page]
    svod_amd.write_pages(k.to(device), v.to(device), pages)
    for now, x in zip(pools, want):
        assert torch.equal(bits(now), x)


# ---- attention_paged: a row in front of its sequence's first token sees no key.
MASKS = {"none": {}, "causal": dict(causal=True), "both sides": dict(window=(33, 65)), "right": dict(window=(0, 500)),
         "causal window": dict(causal=True, window=(40, 0)), "a negative scale": dict(scale=-0.2)}


@pytest.mark.parametrize("dtype,coded", KINDS)
@pytest.mark.parametrize("name", MASKS)
@pytest.mark.parametrize("lens,new,h,splits", [([4, 0, 70], [6, 9, 3], 4, None),            # tiles of 16 rows
                                               ([2, 700, 1], [17, 20, 5], 4, 3),             # split ones, of 32
                                               ([100, 0, 90], [300, 40, 2], 4, None),       # of 128: a tile without a position, one across
                                               ([900, 64], [1100, 200], 4, 4)])             # and split
def test_a_row_without_a_position_sees_no_key(device, lens, new, h, splits, name, dtype, coded):
    opts = MASKS[name]
    case = make(device, [0] * len(new), new, kv_heads=2, d=64, lens=lens, dtype=dtype, coded=coded, seed=len(name))
    q = normal((case.rows, h, 64), dtype, 13, device)
    out = svod_amd.attention_paged(q, case.pages, Attn(splits=splits, **opts))
    want, allowed = ref.attention(case, q, **opts)
    for b, (n, t) in enumerate(zip(lens, new)):
        none = slice(case.starts[b], case.starts[b] + max(0, t - n))
        assert bool((out[none] == 0).all()), b
        want[none] = 0.0  # whatever the mask
    held(out, want, allowed, name)


# ---- attention_paged: numbers out of range, in every form of a launch.
FORMS = {  # contexts, new tokens, query heads, kv heads, D, splits
    "few rows, whole and in parts": ([3000, 40, 500, 9], [1, 2, 1, 3], 4, 2, 64, None),
    "few rows, named splits": ([3000, 40, 500, 9], [1, 2, 1, 3], 4, 2, 128, 5),
    "shares": ([100 + 7 * (i % 40) for i in range(146)] + [9000, 6000, 4000, 7000], [1] * 150, 4, 4, 64, None),
    "32 rows": ([2500, 700, 64, 3], [8, 5, 9, 2], 8, 2, 128, None),
    "chunks": ([300, 0, 77, 500], [200, 150, 1, 30], 4, 2, 64, 1),
    "chunks in parts": ([3000, 700, 64, 2000], [150, 30, 200, 1], 4, 2, 128, None),
    "chunks, named splits": ([3000, 700, 64, 2000], [150, 30, 200, 1], 4, 2, 64, 3),
}


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("bad", ["a length past the table", "a length far past it", "a negative length", "pages that are none", "an end past the rows"])
@pytest.mark.parametrize("name", FORMS)
def test_numbers_out_of_range_stay_with_their_sequence(device, name, bad, coded):
    """One sequence's length, entries or end are wrong: its own rows hold something, those of the others what they should, and nothing beside
    the rows and in the pools is touched."""
    context, new, h, hkv, d, splits = FORMS[name]
    case = make(device, context, new, kv_heads=hkv, d=d, coded=coded, seed=len(name), fill=0.0, rows_after=2, wide=(torch.int64, torch.int64))
    q = normal((case.rows, h, d), BF16, 5, device)
    want, allowed = ref.attention(case, q, causal=True)
    one = len(new) - 1 if bad == "an end past the rows" else 1
    lens, starts, table = case.pages.lens.clone(), case.pages.starts.clone(), case.pages.table.clone()
    limit = table.shape[1] * 16
    if bad == "a length past the table":
        lens[one] = limit + 5
    elif bad == "a length far past it":
        lens[one] = 1 << 60
    elif bad == "a negative length":
        lens[one] = -(1 << 33) + 70
    elif bad == "pages that are none":
        table[one, ::2], table[one, 1::2] = -7, 0x7fffffff
    else:
        starts[one + 1] = case.rows + (1 << 35)
    pages = Pages(case.pages.k, case.pages.v, table, lens, starts, case.pages.scales)
    pools = [case.pages.k, case.pages.v, *(case.pages.scales or ())]
    before = [bits(x).clone() for x in pools]
    guard = torch.full((case.rows + 64, h, d), 5.0, dtype=BF16, device=device)
    out = svod_amd.attention_paged(q, pages, Attn(causal=True, splits=splits), out=guard[32:32 + case.rows])
    assert bool((guard[:32] == 5.0).all()) and bool((guard[32 + case.rows:] == 5.0).all()) and torch.isfinite(out).all()
    want[case.starts[one]:case.starts[one + 1]] = float("nan")  # its own rows
    held(out, want, allowed, name)
    for x, was in zip(pools, before):
        assert torch.equal(bits(x), was)
    # Good numbers in the same places: the call is what it was.
    held(svod_amd.attention_paged(q, case.pages, Attn(causal=True, splits=splits)), *ref.attention(case, q, causal=True))


def test_codes_past_the_other_types_range_are_infinite(device):
    """A pool written from bf16 and read in f16: a row is rounded to it, codes from 65520 on (the middle between its largest value and the
    next) to an infinity, the others in place."""
    codes = torch.arange(0x80, dtype=torch.uint8)[:0x7f].repeat(2, 1)  # both halves: every finite code of one sign, and its negative
    codes[1] |= 0x80
    codes = torch.nn.functional.pad(codes, (0, 1)).expand(1, 1, 8, 2, 128).reshape(1, 1, 16, 128).contiguous()
    e = torch.arange(4, 12).repeat_interleave(2)
    scales = (e + 127).to(torch.uint8).view(1, 1, 16)
    pool, scale = codes.to(device).view(ref.E4M3), scales.to(device).view(ref.E8M0)
    pages = Pages(pool, pool, torch.zeros(1, 1, dtype=torch.int32, device=device), torch.tensor([16], dtype=torch.int32, device=device),
                  scales=(scale, scale))
    stood = codes[0, 0].view(ref.E4M3).double() * torch.pow(2.0, e.double())[:, None]
    want = torch.where(stood.abs() >= 65520, stood.sign() * float("inf"), stood)  # what fits is exact: four significant bits
    for x in svod_amd.read_pages(pages, 16, F16):
        assert torch.equal(x[0, :, 0].double().cpu(), want)
    for x in svod_amd.read_pages(pages, 16, BF16):
        assert torch.equal(x[0, :, 0].double().cpu(), stood)
