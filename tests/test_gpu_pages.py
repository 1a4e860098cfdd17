"""A key/value cache in pages on the device (write_pages, read_pages, attention_paged) against its definitions in 64 bits."""
import numpy as np
import pytest
import torch

import svod_amd
from svod_amd import Attn, KeyMask, Pages
import pages_reference as ref
from pages_reference import E4M3, E8M0, F64, make

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def bits(x):
    return x.detach().cpu().contiguous().view(torch.uint8 if x.element_size() == 1 else torch.int16)


def normal(shape, dtype, seed, device, by=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * by).to(dtype).to(device)


def held(got, want, allowed, what=""):
    got = got.to(F64).cpu()
    rows = ~torch.isnan(want)
    assert torch.isfinite(got[rows]).all(), what
    off = (got - want).abs()[rows]
    bad = off > allowed[rows]
    assert not bad.any(), (what, int(bad.sum()), float((off - allowed[rows]).max()), float((off / allowed[rows].clamp(min=1e-30)).max()))


# ---- attention: (context, new tokens) a sequence, query heads, kv heads, D, page, options.
CASES = {
    "one token of one sequence": ([0], [1], 2, 1, 64, 16, dict(causal=True)),
    "one key each, a page that ends inside a block": ([16, 0, 31, 63, 64, 65], [1] * 6, 4, 2, 128, 16, dict(causal=True)),
    "a step, short and long": ([5, 700, 64, 1, 129], [1] * 5, 16, 8, 128, 32, dict(causal=True)),
    "drafts": ([100, 0, 37, 1000], [5, 3, 7, 1], 20, 20, 64, 16, dict(causal=True)),
    "chunks": ([0, 300, 17, 0], [200, 65, 1, 128], 4, 2, 128, 64, dict(causal=True)),
    "a prompt of several tiles": ([0], [515], 4, 1, 64, 128, dict(causal=True)),
    "sequences without new tokens, and empty ones": ([90, 0, 12, 0], [0, 0, 33, 1], 6, 2, 64, 16, dict(causal=True)),
    "nothing masked": ([50, 0, 200], [3, 70, 1], 8, 2, 128, 16, {}),
    "a group of five": ([33, 400], [9, 60], 15, 3, 64, 16, dict(causal=True)),
    "a group of 71 in tiles of one token": ([40, 130], [2, 3], 71, 1, 64, 16, dict(causal=True)),
    "a group of 128": ([70], [2], 128, 1, 64, 256, dict(causal=True)),
    "a window": ([500, 10, 0], [4, 90, 300], 4, 2, 64, 16, dict(causal=True, window=(70, 0))),
    "a window of the token itself": ([300, 3], [2, 40], 4, 4, 128, 16, dict(causal=True, window=(0, 0))),
    "a window on both sides": ([200, 0], [60, 150], 4, 2, 128, 32, dict(window=(33, 65))),
    "a window past both ends": ([20], [30], 2, 2, 64, 16, dict(window=(1 << 40, 1 << 40))),
    "head size 256": ([100, 5], [1, 40], 4, 2, 256, 16, dict(causal=True)),
    "head size 256, few rows": ([200, 64], [1, 1], 4, 2, 256, 64, dict(causal=True)),
    "pages of 1024": ([1500, 20], [1, 100], 4, 2, 64, 1024, dict(causal=True)),
    "a negative scale": ([90, 200], [1, 2], 4, 2, 64, 16, dict(causal=True, scale=-0.2)),
    "a scale of zero": ([90, 200], [1, 33], 4, 2, 64, 16, dict(causal=True, scale=0.0)),
    "more sequences than lanes": ([i % 37 for i in range(150)], [1 + i % 3 for i in range(150)], 2, 1, 64, 16, dict(causal=True)),
}


@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("kind", ["bf16", "f16", "bf16 e4m3", "f16 e4m3"])
@pytest.mark.parametrize("name", CASES)
def test_attention_over_pages(device, name, kind, splits):
    context, fresh, h, hkv, d, page, opts = CASES[name]
    dtype = F16 if kind.startswith("f16") else BF16
    case = make(device, context, fresh, kv_heads=hkv, d=d, page=page, dtype=dtype, coded="e4m3" in kind, seed=len(name))
    q = normal((case.rows, h, d), dtype, 3, device)
    got = svod_amd.attention_paged(q, case.pages, Attn(splits=splits, **opts))
    torch.cuda.synchronize()
    assert svod_amd.chosen().startswith('Kernel { op: "attention_paged"')
    held(got, *ref.attention(case, q, **opts), name)


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("splits", [None, 2, 1000])
def test_long_sequences_split(device, coded, splits):
    """More blocks than an item may have: the device's own splits, and named ones up to one a block."""
    case = make(device, [4000, 30, 2500], [1, 1, 2], kv_heads=2, d=128, page=16, coded=coded, seed=5)
    q = normal((case.rows, 8, 128), BF16, 4, device, by=2.0)
    got = svod_amd.attention_paged(q, case.pages, Attn(causal=True, splits=splits))
    held(got, *ref.attention(case, q, causal=True))
    assert torch.equal(bits(got), bits(svod_amd.attention_paged(q, case.pages, Attn(causal=True, splits=splits))))


def test_a_chunk_over_a_long_context_splits(device):
    case = make(device, [3000], [150], kv_heads=1, d=64, page=32, seed=6)
    q = normal((case.rows, 2, 64), BF16, 4, device)
    assert svod_amd.attention_paged_workspace(q, case.pages, Attn(causal=True)) > 0
    held(svod_amd.attention_paged(q, case.pages, Attn(causal=True)), *ref.attention(case, q, causal=True))


@pytest.mark.parametrize("coded", [False, True])
def test_lengths_and_starts_of_64_bits(device, coded):
    case = make(device, [40, 0, 300], [2, 20, 1], coded=coded, wide=(torch.int64, torch.int64), seed=8)
    q = normal((case.rows, 4, 64), BF16, 9, device)
    held(svod_amd.attention_paged(q, case.pages, Attn(causal=True)), *ref.attention(case, q, causal=True))


@pytest.mark.parametrize("splits", [None, 2])
@pytest.mark.parametrize("fresh", [[3, 2], [90, 40]])
def test_rows_of_no_sequence_stay_as_they_are(device, fresh, splits):
    """Rows in front of the first sequence and behind the last, as a padded batch or a graph's fixed size leaves them."""
    case = make(device, [300, 500], fresh, seed=10, rows_before=5, rows_after=70)
    q = normal((case.rows, 4, 64), BF16, 11, device)
    q[:5] = float("nan")
    q[case.starts[-1]:] = float("nan")
    out = torch.full_like(q, 7.0)
    svod_amd.attention_paged(q, case.pages, Attn(causal=True, splits=splits), out=out)
    assert bool((out[:5] == 7.0).all()) and bool((out[case.starts[-1]:] == 7.0).all())
    want, allowed = ref.attention(case, torch.where(torch.isnan(q), 0.0, q), causal=True)
    held(out, want, allowed)


def test_a_length_short_of_its_new_rows(device):
    """Fewer tokens than rows: the first rows have no position, see nothing and are not stored."""
    case = make(device, [0, 0], [6, 9], lens=[4, 0], seed=12)
    q = normal((case.rows, 2, 64), BF16, 13, device)
    out = svod_amd.attention_paged(q, case.pages, Attn(causal=True))
    assert bool((out[:2] == 0).all()) and bool((out[6:] == 0).all())
    want, allowed = ref.attention(case, q, causal=True)
    held(out, want, allowed)
    k = normal((case.rows, 2, 64), BF16, 14, device)
    before = case.pages.k.clone()
    svod_amd.write_pages(k, k, case.pages)
    rows = case.pages.k[int(case.table[0, 0]), :, :4]
    assert torch.equal(bits(rows), bits(k[2:6].transpose(0, 1)))
    before[int(case.table[0, 0]), :, :4] = rows
    assert torch.equal(bits(case.pages.k), bits(before))


def test_bad_lengths_starts_and_pages_stay_inside(device):
    """Device data that no host check sees: held inside the table, the packed rows and the pool, with a result that is wrong
    or left out and nothing beside it touched."""
    case = make(device, [40, 300, 20], [2, 3, 4], seed=15, fill=0.0)
    q = normal((case.rows, 4, 64), BF16, 16, device)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=device)
    wild = torch.full_like(case.pages.table, -5)
    wild[:, ::2] = 0x7ffffff0
    for change in (dict(table=wild), dict(lens=i32(-3, 1 << 30, 20)), dict(lens=i64(1 << 40, -(1 << 40), 3)),
                   dict(starts=i32(-9, 4, 2, 1 << 30)), dict(starts=i64(0, 9, 0, 1 << 50)), dict(starts=i32(9, 9, 9, 9))):
        fields = {**case.pages.__dict__, **change}
        pages = Pages(**{**fields, "k": fields["k"].clone(), "v": fields["v"].clone()})
        guard = torch.full((case.rows + 64, 4, 64), 5.0, dtype=BF16, device=device)
        out = svod_amd.attention_paged(q, pages, Attn(causal=True), out=guard[32:32 + case.rows])
        assert bool((guard[:32] == 5.0).all()) and bool((guard[32 + case.rows:] == 5.0).all()) and torch.isfinite(out).all()
        svod_amd.write_pages(q[:, :2].contiguous(), q[:, 2:].contiguous(), pages)
        k, v = svod_amd.read_pages(pages, 50)
        assert torch.isfinite(k).all() and torch.isfinite(v).all()


# ---- write and read.
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("kind", ["bf16", "f16", "bf16 e4m3", "f16 e4m3"])
def test_written_and_read_back(device, kind, page, d):
    dtype = F16 if kind.startswith("f16") else BF16
    coded = "e4m3" in kind
    case = make(device, [0, 13, 100, 0, 31], [1, 50, 3, 0, 17], kv_heads=3, d=d, page=page, dtype=dtype, coded=coded, seed=page + d,
                rows_before=2, rows_after=3)
    k, v = (normal((case.rows, 3, d), dtype, s, "cpu", by=4.0) for s in (20, 21))
    before = [x.clone() for x in (case.pages.k.view(torch.uint8), case.pages.v.view(torch.uint8))]
    svod_amd.write_pages(k.to(device), v.to(device), case.pages)
    assert svod_amd.chosen().startswith('Kernel { op: "write_pages"')
    written = torch.zeros(case.k.shape[0], page, dtype=torch.bool)
    for row, b, at in case.places():
        i, r = int(case.table[b, at // page]), at % page
        written[i, r] = True
        for x, pool in ((k, case.k), (v, case.v)):
            pool[i, :, r] = ref.quantised(x[row])[0] if coded else x[row].to(F64)
    for pool, was in zip((case.pages.k, case.pages.v), before):  # the others are as they were
        now = pool.view(torch.uint8).cpu()
        assert torch.equal(now.transpose(1, 2)[~written], was.cpu().transpose(1, 2)[~written])
    for tokens in (1, 40, 130):
        got = svod_amd.read_pages(case.pages, tokens, dtype)
        assert svod_amd.chosen().startswith('Kernel { op: "read_pages"')
        for x, which in zip(got, ("k", "v")):
            want = torch.zeros(len(case.lens), tokens, 3, d, dtype=F64)
            for b, n in enumerate(case.lens):
                want[b, :min(n, tokens)] = case.tokens(which, b)[:tokens]
            assert torch.equal(x.to(F64).cpu(), want)  # the codes' values are the type's own


def edges(dtype):
    """Rows at the borders of a scale and of a code, [rows, 64]."""
    f = torch.finfo(dtype)
    rows = []
    for amax in (448.0, 450.0, 1.75, 1.7578125, 3.5, 2.0 ** -7, f.tiny, f.smallest_normal * 448, f.max, f.max / 2, 57344.0, 57376.0, 0.0):
        amax = float(torch.tensor(amax, dtype=F64).to(dtype).to(F64))
        if not np.isfinite(amax) or amax > f.max:
            continue
        # Ties between codes, the values next to them, and what lies below the least code.
        parts = [amax * x for x in (1, -1, 17 / 32, 19 / 32, 1 / 448, 1.5 / 448, 2.0 ** -10 / 448, 2.0 ** -9 / 448, 3 * 2.0 ** -10 / 448, 31 / 32)]
        rows.append(parts + [amax * (i / 54) * (-1) ** i for i in range(54)])
    x = torch.tensor(rows, dtype=F64).to(dtype)
    bad = x[:3].clone()
    bad[0, 3], bad[1, 5], bad[2, 0] = float("inf"), float("nan"), -float("inf")
    tiny = torch.zeros(2, 64, dtype=dtype)
    tiny[0, 7], tiny[1, 0] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps, -0.0
    none = torch.full((1, 64), float("nan"), dtype=dtype)
    return torch.cat([x, bad, tiny, none])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_quantised_at_the_borders(device, dtype):
    x = edges(dtype)
    n = x.shape[0]
    case = make(device, [0], [n], kv_heads=1, d=64, page=64, dtype=dtype, coded=True, seed=1, fill=0.0)
    svod_amd.write_pages(x[:, None].to(device), -x[:, None].to(device), case.pages)
    want, e = ref.quantised(x)
    at = int(case.table[0, 0])
    codes = case.pages.k[at, 0, :n].to(torch.float32).cpu().to(F64)
    assert torch.equal(case.pages.scales[0][at, 0, :n].view(torch.uint8).cpu().long() - 127, e)
    stood = codes * torch.pow(2.0, e.to(F64))[:, None]
    assert torch.equal(torch.isnan(stood), ~torch.isfinite(x))
    assert torch.equal(torch.nan_to_num(stood), torch.nan_to_num(want))
    k, v = svod_amd.read_pages(case.pages, n, dtype)
    assert torch.equal(torch.isnan(k[0, :, 0]).cpu(), ~torch.isfinite(x)) and not torch.isinf(k).any()
    fits = want.abs() >= torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # what the type has no value for is zero
    assert torch.equal(torch.where(fits, k[0, :, 0].to(F64).cpu(), 0.0), torch.where(fits, want, 0.0))
    assert torch.equal(torch.nan_to_num(v), torch.nan_to_num(-k))
    # Half a step of e4m3, or of its least one.
    off = (torch.nan_to_num(stood) - torch.nan_to_num(x.to(F64), posinf=0.0, neginf=0.0)).abs()
    assert bool((off[torch.isfinite(x)] <= torch.maximum(x.to(F64).abs() * ref.half_step(E4M3),
                                                         torch.pow(2.0, e.to(F64) - 10)[:, None].expand_as(x))[torch.isfinite(x)]).all())


def test_every_code_is_read_as_what_it_stands_for(device):
    """All 256 codes at every scale the writer makes, in bf16 exactly (f16 where it holds them)."""
    page = 64
    scales = torch.arange(10, 248, dtype=torch.uint8)
    count = -(-len(scales) // page)
    codes = torch.arange(256, dtype=torch.uint8).expand(count, 1, page, 256).contiguous()
    held_scales = torch.full((count * page,), 127, dtype=torch.uint8)
    held_scales[:len(scales)] = scales
    pages = Pages(codes.to(device).view(E4M3), codes.to(device).view(E4M3), torch.arange(count, dtype=torch.int32, device=device)[None],
                  torch.tensor([count * page], dtype=torch.int32, device=device),
                  scales=(held_scales.view(count, 1, page).to(device).view(E8M0),) * 2)
    want = codes[0, 0, 0].view(E4M3).float().to(F64)[None] * torch.pow(2.0, held_scales.to(F64) - 127)[:, None]
    k, _ = svod_amd.read_pages(pages, count * page)
    # (Codes from 256 on at 2^120, which the writer does not make, are 2^128 and more: past bf16's largest, 2^128 - 2^120.)
    fits = want.abs() <= torch.finfo(BF16).max
    assert int((~fits & ~torch.isnan(want)).sum()) == 2 * 7 and bool((want[~fits & ~torch.isnan(want)].abs() >= 2.0 ** 128).all())
    assert torch.equal(k[0, :, 0].to(F64).cpu()[fits], want[fits])
    assert torch.equal(torch.isnan(k[0, :, 0]).cpu(), torch.isnan(want))
    k, _ = svod_amd.read_pages(pages, count * page, F16)
    fits = (want.abs() <= 65504) & (want.abs() >= 2.0 ** -14)
    assert torch.equal(k[0, :, 0].to(F64).cpu()[fits], want[fits])


# ---- as they are used together.
@pytest.mark.parametrize("coded", [False, True])
def test_a_prompt_then_tokens(device, coded):
    """Prompts in chunks, then single tokens, through prologue, cache and attention: each step's result against attention over
    the same tokens in rows."""
    h, hkv, d, page = 4, 2, 64, 16
    lens, steps = [0, 0, 0], [[70, 33, 5], [64, 0, 12], [1, 1, 1], [1, 1, 1]]
    total = [sum(s[b] for s in steps) for b in range(3)]
    counts = [-(-n // page) for n in total]
    table = torch.zeros(3, max(counts), dtype=torch.int32)
    ids = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(2)).tolist()
    for b in range(3):
        table[b, :counts[b]] = torch.tensor([ids.pop() for _ in range(counts[b])])
    shape = (sum(counts), hkv, page, d)
    pool = lambda: (torch.zeros(shape, dtype=torch.uint8, device=device).view(E4M3) if coded else torch.zeros(shape, dtype=BF16, device=device))
    scales = tuple(torch.zeros(shape[:3], dtype=torch.uint8, device=device).view(E8M0) for _ in range(2)) if coded else None
    pages = Pages(pool(), pool(), table.to(device), torch.zeros(3, dtype=torch.int32, device=device),
                  torch.zeros(4, dtype=torch.int32, device=device), scales)
    for n, fresh in enumerate(steps):
        rows = sum(fresh)
        qkv = normal((1, rows, (h + 2 * hkv) * d), BF16, 30 + n, device)
        q, k, v = svod_amd.heads(qkv, svod_amd.Qkv(h, hkv, d))
        lens = [a + b for a, b in zip(lens, fresh)]
        pages.lens.copy_(torch.tensor(lens))
        pages.starts.copy_(torch.tensor([0, *np.cumsum(fresh).tolist()]))
        svod_amd.write_pages(k[0], v[0], pages)
        got = svod_amd.attention_paged(q[0], pages, Attn(causal=True))
        kr, vr = svod_amd.read_pages(pages, max(lens))
        at = 0
        for b, t in enumerate(fresh):
            if t == 0:
                continue
            # A causal call counts its queries from the first key: the earlier tokens stand in front as queries of zeros.
            padded = torch.cat([torch.zeros(1, lens[b] - t, h, d, dtype=BF16, device=device), q[:, at:at + t]], 1)
            want = svod_amd.attention(padded, kr[b:b + 1, :lens[b]].contiguous(), vr[b:b + 1, :lens[b]].contiguous(), Attn(causal=True))
            # Two roundings of the same sums to bf16, and of the probabilities: u each, of values up to the rows' largest.
            most = float(vr[b].abs().max())
            assert float((got[at:at + t].float() - want[0, -t:].float()).abs().max()) <= 4 * 2.0 ** -8 * most
            at += t


def test_read_pages_feeds_attention(device):
    case = make(device, [200, 77], [1, 1], kv_heads=2, d=64, seed=40)
    q = normal((2, 4, 64), BF16, 41, device)
    k, v = svod_amd.read_pages(case.pages, 201)
    by_rows = svod_amd.attention(q[:, None].contiguous(), k, v, Attn(keys=KeyMask.lens(case.pages.lens)))
    want, allowed = ref.attention(case, q, causal=True)
    held(by_rows[:, 0], want, allowed)
    held(svod_amd.attention_paged(q, case.pages, Attn(causal=True)), want, allowed)


def test_a_replayed_step_follows_its_lengths(device):
    """One captured graph of a step: lengths, starts, table and operands change between its replays."""
    h, hkv, d, page, batch = 4, 2, 64, 16, 4
    case = make(device, [500, 400, 300, 600], [1, 1, 1, 1], kv_heads=hkv, d=d, page=page, seed=50)
    q, k, v = (normal((batch, n, d), BF16, 51 + n, device) for n in (h, hkv, hkv))
    out = torch.empty_like(q)
    opts = Attn(causal=True)
    ws = torch.empty(svod_amd.attention_paged_workspace(q, case.pages, opts), dtype=torch.uint8, device=device)

    def step():
        svod_amd.write_pages(k, v, case.pages)
        svod_amd.attention_paged(q, case.pages, opts, out, ws)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for n, lens in enumerate(([500, 1, 300, 2], [17, 401, 64, 601], [501, 401, 301, 601])):
        case.pages.lens.copy_(torch.tensor(lens))
        for x, s in ((q, 60 + n), (k, 70 + n), (v, 80 + n)):
            x.copy_(normal(tuple(x.shape), BF16, s, device))
        ws.fill_(0xff)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        out.fill_(0)
        step()
        assert torch.equal(bits(replayed), bits(out))
        case.lens[:] = lens
        for row, b, at in case.places():
            case.k[int(case.table[b, at // page]), :, at % page] = k[row].to(F64).cpu()
            case.v[int(case.table[b, at // page]), :, at % page] = v[row].to(F64).cpu()
        held(replayed, *ref.attention(case, q, causal=True))


def test_two_streams_at_once(device):
    cases = [make(device, [700 + 50 * i, 90], [1, 3], kv_heads=2, d=128, seed=90 + i) for i in range(2)]
    qs = [normal((c.rows, 4, 128), BF16, 95 + i, device) for i, c in enumerate(cases)]
    want = [svod_amd.attention_paged(q, c.pages, Attn(causal=True)) for q, c in zip(qs, cases)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(svod_amd.attention_paged(qs[i], cases[i].pages, Attn(causal=True)))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(bits(x), bits(want[i]))
