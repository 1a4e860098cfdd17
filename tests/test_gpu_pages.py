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


# ---- calls of every form, at their borders.
def ragged(count, seed, least, most):
    r = np.random.default_rng(seed)
    return [int(x) for x in r.integers(least, most + 1, count)]


def both(device, case, h, opts, seed=3, by=1.0):
    """The call's result held to the reference, and the same bits from a second call."""
    q = normal((case.rows, h, case.k.shape[3]), case.dtype, seed, device, by)
    got = svod_amd.attention_paged(q, case.pages, Attn(**opts))
    held(got, *ref.attention(case, q, **{k: v for k, v in opts.items() if k != "splits"}))
    assert torch.equal(bits(got), bits(svod_amd.attention_paged(q, case.pages, Attn(**opts))))
    return svod_amd.chosen()


KINDS = [(BF16, False), (F16, False), (BF16, True), (F16, True)]


@pytest.mark.parametrize("dtype,coded", KINDS)
@pytest.mark.parametrize("window", [None, (70, 0), (200, 3)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_chunks_beside_single_tokens(device, d, window, dtype, coded):
    """More sequences than lanes, a few with chunks between those of one to five tokens: two tile forms in one launch."""
    context, fresh = ragged(71, d, 0, 300), ragged(71, d + 1, 0, 5)
    for b, n in ((3, 150), (40, 129), (66, 128), (70, 31)):
        fresh[b] = n
    case = make(device, context, fresh, kv_heads=1, d=d, page=32, dtype=dtype, coded=coded, seed=d)
    assert "rows: 128" in both(device, case, 8, dict(causal=True, window=window))


@pytest.mark.parametrize("dtype,coded", KINDS)
def test_a_long_sequence_among_many_is_split(device, dtype, coded):
    """Tiles for more than half of the places and one sequence far longer than the others: of 128 rows its own alone is split."""
    fresh = [128] * 70 + [1, 130]
    context = ragged(70, 5, 0, 64) + [20000, 9000]
    case = make(device, context, fresh, kv_heads=2, d=64, page=64, dtype=dtype, coded=coded, seed=9)
    q = normal((case.rows, 4, 64), dtype, 3, device)
    assert svod_amd.attention_paged_workspace(q, case.pages, Attn(causal=True)) > 0
    assert "rows: 128" in both(device, case, 4, dict(causal=True))


@pytest.mark.parametrize("dtype,coded", KINDS)
@pytest.mark.parametrize("d,h,hkv,fresh", [(64, 4, 4, 1), (128, 8, 4, 1), (64, 8, 4, 5), (128, 16, 4, 6)])
def test_shares_of_many_ragged_sequences(device, d, h, hkv, fresh, dtype, coded):
    """Few rows a sequence, more tiles than half of the places, lengths that differ much: every place takes an even share of all
    blocks, which begins and ends inside tiles, and tiles lie in the shares of one to many places."""
    context = ragged(150, d, 0, 150)
    context[7], context[80], context[149] = 9000, 4000, 6000
    case = make(device, context, [1 + b % fresh for b in range(150)], kv_heads=hkv, d=d, page=16, dtype=dtype, coded=coded, seed=d + h)
    assert "rows: 128" not in both(device, case, h, dict(causal=True))


@pytest.mark.parametrize("group,tokens,d", [(1, 16, 64), (1, 17, 64), (16, 1, 128), (17, 1, 128), (32, 1, 64), (33, 1, 64), (4, 8, 128),
                                            (4, 9, 128), (5, 3, 128), (16, 1, 256), (17, 1, 256), (127, 1, 128)])
def test_rows_at_the_forms_borders(device, group, tokens, d):
    case = make(device, [333, 0, 64, 1000], [tokens] * 4, kv_heads=1, d=d, page=16, seed=group)
    both(device, case, group, dict(causal=True))
    both(device, case, group, dict(causal=True, splits=4))


@pytest.mark.parametrize("coded", [False, True])
def test_one_very_long_sequence(device, coded):
    case = make(device, [150_000], [2], kv_heads=1, d=64, page=256, coded=coded, seed=2)
    both(device, case, 3, dict(causal=True))
    case.pages.lens[0] = case.lens[0] = 149_999
    both(device, case, 3, dict(causal=True, window=(70_000, 0)))


def test_more_splits_than_a_merge_takes_at_once(device):
    """A state a block: a tile of several hundred, of few rows and of 128."""
    for fresh in (1, 130):
        case = make(device, [20_000, 70], [fresh, 1], kv_heads=1, d=64, page=64, seed=fresh)
        both(device, case, 4, dict(causal=True, splits=400))


@pytest.mark.parametrize("coded", [False, True])
@pytest.mark.parametrize("fresh", [[1, 2, 1], [70, 90, 40]])
def test_pages_in_front_of_the_window_are_not_read(device, coded, fresh):
    """What a sequence's window has left it may give away: the table's entries there point at a page of NaN, or at none."""
    window, page = (100, 0), 32
    case = make(device, [500, 37, 1000], fresh, kv_heads=2, d=64, page=page, coded=coded, seed=4)
    q = normal((case.rows, 32, 64), BF16, 5, device)
    opts = Attn(causal=True, window=window)
    want = svod_amd.attention_paged(q, case.pages, opts)
    held(want, *ref.attention(case, q, causal=True, window=window))
    spare = next(i for i in range(case.k.shape[0]) if not bool((case.table == i).any()))
    for x in (case.pages.k, case.pages.v):
        x[spare].view(torch.uint8 if coded else torch.int16).fill_(0x7f if coded else 0x7fff)
    for b, n in enumerate(case.lens):
        gone = max(0, n - fresh[b] - window[0]) // page
        case.pages.table[b, :gone] = spare
        case.pages.table[b, :gone:3] = -1
    case.pages.table[1, -1] = 0x7fffffff
    assert torch.equal(bits(want), bits(svod_amd.attention_paged(q, case.pages, opts)))


@pytest.mark.parametrize("coded", [False, True])
def test_pools_past_4_gib(device, coded):
    """Offsets that pass 32 bits: the pages at both ends of pools of 4.6 GiB."""
    page, d, hkv = 64, 128, 8
    count = (9 << 29) // (page * d * hkv * (1 if coded else 2)) + 3
    case = make(device, [200, 70, 0], [3, 1, 40], kv_heads=hkv, d=d, page=page, coded=coded, seed=6, fill=0.0)
    small = case.pages
    ids = torch.arange(case.k.shape[0])
    at = torch.where(ids % 2 == 0, ids, count - 1 - ids)  # where the small pool's pages stand in the large one
    pools = [torch.empty((count, *x.shape[1:]), dtype=torch.uint8 if coded else BF16, device=device) for x in (small.k, small.v)]
    for pool, x in zip(pools, (small.k, small.v)):
        for i, to in enumerate(at.tolist()):
            pool[to].copy_(x[i].view(pool.dtype))
    assert pools[0].numel() * pools[0].element_size() > 1 << 32
    scales = None
    if coded:
        scales = tuple(torch.empty((count, hkv, page), dtype=torch.uint8, device=device) for _ in range(2))
        for s, x in zip(scales, small.scales):
            for i, to in enumerate(at.tolist()):
                s[to].copy_(x[i].view(torch.uint8))
        pools, scales = [p.view(E4M3) for p in pools], tuple(s.view(E8M0) for s in scales)
    table = small.table.clone().cpu()
    used = (table >= 0) & (table < len(ids))
    table[used] = at[table[used].long()].to(torch.int32)
    large = Pages(pools[0], pools[1], table.to(device), small.lens, small.starts, scales)
    q, k = normal((case.rows, 16, d), BF16, 8, device), normal((case.rows, hkv, d), BF16, 9, device, by=3.0)
    for step in range(2):
        got, want = (svod_amd.attention_paged(q, p, Attn(causal=True)) for p in (large, small))
        assert torch.equal(bits(got), bits(want))
        for a, b in zip(svod_amd.read_pages(large, 210), svod_amd.read_pages(small, 210)):
            assert torch.equal(bits(a), bits(b))
        for p in (large, small):
            svod_amd.write_pages(k, -k, p)


@pytest.mark.parametrize("dtype,coded", KINDS)
def test_many_rows_are_written_as_few_are(device, dtype, coded):
    """Large calls take four heads a wave, here with one over: the same pages as sequence by sequence, and unlike values too."""
    hkv, d, page = 13, 128, 64
    fresh = [1500, 1, 700, 0, 803]
    big = make(device, [0, 5, 100, 9, 64], fresh, kv_heads=hkv, d=d, page=page, dtype=dtype, coded=coded, seed=7, fill=0.0, rows_before=3, rows_after=2)
    k, v = (normal((big.rows, hkv, d), dtype, s, device, by=3.0) for s in (1, 2))
    k[::7] *= 2.0 ** -12
    k[11, :, 5], k[12, 3, 9], v[13, 12, 127] = float("inf"), float("nan"), -float("inf")
    v[::5] *= 1000.0
    one = Pages(big.pages.k.clone(), big.pages.v.clone(), big.pages.table, big.pages.lens, big.pages.starts,
                tuple(x.clone() for x in big.pages.scales) if coded else None)
    svod_amd.write_pages(k, v, big.pages)
    for b in range(5):
        s, e = big.starts[b], big.starts[b + 1]
        for at in range(s, e, 400):  # the sequence's rows a few hundred at a time
            to = min(e, at + 400)
            lens = torch.tensor([big.lens[b] - (e - to)], dtype=torch.int32, device=device)
            starts = torch.tensor([0, to - at], dtype=torch.int32, device=device)
            svod_amd.write_pages(k[at:to].contiguous(), v[at:to].contiguous(),
                                 Pages(one.k, one.v, one.table[b:b + 1].contiguous(), lens, starts, one.scales))
    pairs = [(big.pages.k, one.k), (big.pages.v, one.v), *(zip(big.pages.scales, one.scales) if coded else ())]
    for a, b in pairs:
        assert torch.equal(bits(a), bits(b))


def test_a_shared_prefix(device):
    """Two sequences over the same first pages, and one that is there twice."""
    case = make(device, [640, 700, 64], [1, 1, 1], kv_heads=2, d=64, page=64, seed=3)
    case.table[1, :10] = case.table[0, :10]
    case.pages.table.copy_(case.table)
    both(device, case, 4, dict(causal=True))
    twice = Pages(**{**case.pages.__dict__, "table": case.pages.table[[0, 0, 0]].contiguous(),
                     "lens": case.pages.lens[[0, 0, 0]].contiguous()})
    q = normal((1, 4, 64), BF16, 4, device).expand(3, 4, 64).contiguous()
    got = svod_amd.attention_paged(q, twice, Attn(causal=True))
    assert torch.equal(bits(got[0]), bits(got[1])) and torch.equal(bits(got[0]), bits(got[2]))
    k, _ = svod_amd.read_pages(twice, 641)
    assert torch.equal(bits(k[0]), bits(k[1])) and torch.equal(bits(k[0]), bits(k[2]))


def test_two_graphs_and_eager_calls_on_one_workspace(device):
    """Two captured steps of unlike forms and a call of its own use one workspace in turn; lengths change between the replays, and
    once the starts are not ascending: what that leaves in the workspace costs the next replay nothing."""
    opts = Attn(causal=True)
    cases = [make(device, [2000, 900, 50], [1, 1, 2], kv_heads=2, d=128, page=16, seed=60),
             make(device, [100] * 97 + [3000, 2500, 40], [1] * 100, kv_heads=8, d=128, page=16, seed=61),
             make(device, [3000, 20], [140, 1], kv_heads=1, d=128, page=16, seed=62)]
    heads = (4, 16, 8)
    qs = [normal((c.rows, h, 128), BF16, 63 + i, device) for i, (c, h) in enumerate(zip(cases, heads))]
    ws = torch.empty(max(svod_amd.attention_paged_workspace(q, c.pages, opts) for q, c in zip(qs, cases)), dtype=torch.uint8, device=device)
    assert all(svod_amd.attention_paged_workspace(q, c.pages, opts) > 0 for q, c in zip(qs, cases))
    outs = [torch.empty_like(q) for q in qs]
    run = lambda i: svod_amd.attention_paged(qs[i], cases[i].pages, opts, outs[i], ws)
    stream, graphs = torch.cuda.Stream(), []
    with torch.cuda.stream(stream):
        for i in range(3):
            run(i)
    torch.cuda.synchronize()
    for i in range(3):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            run(i)
    first = [(c.pages.lens.clone(), c.pages.starts.clone()) for c in cases]
    for turn in range(6):
        for c, (lens, starts) in zip(cases, first):
            c.pages.lens.copy_(lens if turn % 2 == 0 else (lens * (turn + 1)) // (turn + 3))
            c.pages.starts.copy_(starts)
            if turn == 3:  # wrong: some tiles more than there are rows
                c.pages.starts[1::2] = 0
                c.pages.starts[::2] = c.rows
        for i in (0, 1, 2, 1, 0):
            outs[i].fill_(9.0)
            graphs[i].replay()
            torch.cuda.synchronize()
            if turn == 3:
                continue
            got = outs[i].clone()
            run((i + 1) % 3)  # and the workspace holds something else
            want = svod_amd.attention_paged(qs[i], cases[i].pages, opts)
            assert torch.equal(bits(got), bits(want)), (turn, i)
            cases[i].lens[:] = cases[i].pages.lens.cpu().tolist()
            if turn < 2:
                held(got, *ref.attention(cases[i], qs[i], causal=True))


def test_a_workspace_of_any_content_and_size(device):
    opts = Attn(causal=True)
    for case, h in ((make(device, [2000, 900, 50], [1, 1, 2], kv_heads=2, d=64, page=16, seed=60), 4),
                    (make(device, [3000, 20], [140, 1], kv_heads=1, d=64, page=16, seed=62), 8)):
        q = normal((case.rows, h, 64), BF16, 1, device)
        need = svod_amd.attention_paged_workspace(q, case.pages, opts)
        want = svod_amd.attention_paged(q, case.pages, opts)
        for fill in (0, 0xff, 0x7f, 1):
            ws = torch.full((need + 256,), fill, dtype=torch.uint8, device=device)
            assert torch.equal(bits(want), bits(svod_amd.attention_paged(q, case.pages, opts, None, ws[:need])))
            assert bool((ws[need:] == fill).all())
        small = svod_amd.attention_paged(q, case.pages, opts, None, ws[:need - 16])  # the keys stay whole
        assert torch.equal(bits(small), bits(svod_amd.attention_paged(q, case.pages, Attn(causal=True, splits=1))))


def test_left_to_the_graph(device):
    """What a device has no kernel for, named."""
    case = make(device, [300], [2], kv_heads=1, d=64, page=16)
    q = normal((2, 4, 64), BF16, 1, device)
    call = lambda p, opts, q=q, **kw: svod_amd.attention_paged(q, p, opts, **kw)

    def why(f):
        with pytest.raises(svod_amd.GraphFallback) as e:
            f()
        return e.value.why

    some = torch.zeros(1, dtype=torch.int32, device=device)
    for opts in (Attn(keys=KeyMask.lens(some)), Attn(bias=torch.zeros(1, 4, 2, 302, dtype=torch.float32, device=device))):
        assert why(lambda: call(case.pages, opts)) == svod_amd.Fallback.Config
    named = Attn(causal=True, splits=3)
    need = svod_amd.attention_paged_workspace(q, case.pages, named)
    lent = torch.empty(need, dtype=torch.uint8, device=device)
    assert why(lambda: call(case.pages, named, workspace=lent[:need - 16])) == svod_amd.Fallback.Config
    call(case.pages, named, workspace=lent)
    shape = lambda n, page, d: Pages(*(torch.zeros(n, 1, page, d, dtype=BF16, device=device) for _ in range(2)), case.pages.table,
                                     case.pages.lens, case.pages.starts)
    for page, d in ((8, 64), (24, 64), (2048, 64), (16, 32), (16, 96)):
        p, x = shape(40, page, d), torch.zeros(2, 1, d, dtype=BF16, device=device)
        assert why(lambda: call(p, None, x)) == svod_amd.Fallback.Shape
        assert why(lambda: svod_amd.write_pages(x, x, p)) == svod_amd.Fallback.Shape
        assert why(lambda: svod_amd.read_pages(p, 5)) == svod_amd.Fallback.Shape
    assert why(lambda: call(case.pages, None, normal((2, 129, 64), BF16, 1, device))) == svod_amd.Fallback.Shape
    assert why(lambda: call(case.pages, None, q[:0])) == svod_amd.Fallback.Shape
    with pytest.raises(svod_amd.OpError) as e:  # what is written may not be read
        call(case.pages, None, out=q)
    assert e.value.kind == "Launch"  # as every op answers parameters that share memory


def test_operands_that_the_host_holds_are_refused(device):
    """Lengths, starts and tables are easily kept on the host: no kernel follows an address there."""
    case = make(device, [300, 40], [2, 1], kv_heads=1, d=64, page=16, coded=True)
    q, k = normal((3, 4, 64), BF16, 1, device), normal((3, 1, 64), BF16, 2, device)
    fields = case.pages.__dict__

    def refused(f):
        with pytest.raises(svod_amd.OpError) as e:
            f()
        assert e.value.kind == "Argument", e.value

    moved = [Pages(**{**fields, n: fields[n].cpu()}) for n in ("k", "v", "table", "lens", "starts")]
    moved.append(Pages(**{**fields, "scales": (fields["scales"][0], fields["scales"][1].cpu())}))
    for p in moved:
        refused(lambda: svod_amd.attention_paged(q, p, Attn(causal=True)))
        refused(lambda: svod_amd.write_pages(k, k, p))
        refused(lambda: svod_amd.read_pages(p, 7))
    refused(lambda: svod_amd.attention_paged(q.cpu(), case.pages))
    refused(lambda: svod_amd.attention_paged(q, case.pages, out=torch.empty(3, 4, 64, dtype=BF16)))
    refused(lambda: svod_amd.attention_paged(q, case.pages, workspace=torch.empty(1 << 20, dtype=torch.uint8)))
    refused(lambda: svod_amd.write_pages(k, k.cpu(), case.pages))
    everything = Pages(**{n: (tuple(y.cpu() for y in x) if n == "scales" else x.cpu()) for n, x in fields.items()})
    refused(lambda: svod_amd.attention_paged(q.cpu(), everything))
    refused(lambda: svod_amd.write_pages(k.cpu(), k.cpu(), everything))
    refused(lambda: svod_amd.read_pages(everything, 7))
    lent = torch.empty(2, 1 << 20, dtype=torch.uint8, device=device)
    refused(lambda: svod_amd.attention_paged(q, case.pages, workspace=lent[:, ::2]))


def test_on_the_stream_of_the_moment(device):
    """Operands made on a stream of their own just before the calls, which follow on it."""
    case = make(device, [900, 40], [1, 30], kv_heads=2, d=64, page=16, seed=12)
    q0 = normal((case.rows, 4, 64), BF16, 1, device)
    kv = normal((case.rows, 2, 64), BF16, 2, device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        busy = torch.randn(4096, 4096, device=device)
        for _ in range(20):
            busy = busy @ busy * 1e-3
        q = q0 * 2.0 + busy[0, 0].nan_to_num(0.0, 0.0, 0.0).to(BF16) * 0.0
        svod_amd.write_pages(kv, kv, case.pages)
        got = svod_amd.attention_paged(q, case.pages, Attn(causal=True))
        k, _ = svod_amd.read_pages(case.pages, 901)
    stream.synchronize()
    for row, b, at in case.places():
        case.k[int(case.table[b, at // 16]), :, at % 16] = kv[row].to(F64).cpu()
        case.v[int(case.table[b, at // 16]), :, at % 16] = kv[row].to(F64).cpu()
    held(got, *ref.attention(case, q0 * 2.0, causal=True))
    assert torch.equal(k[0].to(F64).cpu(), case.tokens("k", 0))


@pytest.mark.parametrize("seed", range(60))
def test_seeded_sweep(device, seed):
    """Calls that draw everything at once: batch, lengths, heads, pages, types, masks, splits, rows around the sequences."""
    r = np.random.default_rng(1000 + seed)
    pick = lambda *x: x[int(r.integers(len(x)))]
    d, page, dtype, coded = pick(64, 128, 256), pick(16, 32, 128, 1024), pick(BF16, F16), pick(False, True)
    hkv, group = pick(1, 2, 3, 8), pick(1, 2, 4, 5, 8, 20)
    batch, most = pick((1, 6000), (3, 2500), (20, 500), (90, 150))
    new = pick(1, 1, 4, 40, 200)
    if batch * new > 1500:
        new = 4
    context = [int(x) for x in np.exp(r.uniform(0, np.log(most), batch))]
    fresh = [int(r.integers(0, new + 1)) if r.random() < 0.8 else min(1, new) for _ in range(batch)]
    fresh[int(r.integers(batch))] = max(1, new)
    causal = bool(r.random() < 0.8)
    window = None if r.random() < 0.6 else (int(r.integers(0, 400)), int(r.integers(0, 100)) if not causal else 0)
    opts = dict(causal=causal, window=window, scale=pick(None, 0.05, -0.03))
    case = make(device, context, fresh, kv_heads=hkv, d=d, page=page, dtype=dtype, coded=coded, seed=seed,
                rows_before=pick(0, 3), rows_after=pick(0, 33), wide=(pick(torch.int32, torch.int64), pick(torch.int32, torch.int64)),
                columns=pick(None, 200 + 6400 // page))
    q = normal((case.rows, hkv * group, d), dtype, seed, device)
    splits = pick(None, None, None, 1, 2, 7)
    out = torch.full_like(q, 3.0)
    svod_amd.attention_paged(q, case.pages, Attn(splits=splits, **opts), out=out)
    held(out, *ref.attention(case, q, **opts), (seed, svod_amd.chosen()))
    s, e = case.starts[0], case.starts[-1]
    assert bool((out[:s] == 3.0).all()) and bool((out[e:] == 3.0).all())
    again = torch.full_like(q, 3.0)
    svod_amd.attention_paged(q, case.pages, Attn(splits=splits, **opts), out=again)
    assert torch.equal(bits(out), bits(again))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("fresh,h", [(5, 2), (40, 2), (200, 8)])
def test_keys_that_a_row_does_not_see_may_hold_anything(device, fresh, h, bad):
    """A new token's key that is no number: the rows in front of it, in its own tile and block, are what they were; a row behind sees it."""
    case = make(device, [77], [fresh], kv_heads=1, d=64, page=16, seed=21)
    q = normal((fresh, h, 64), BF16, 22, device)
    want = svod_amd.attention_paged(q, case.pages, Attn(causal=True))
    at = 77 + fresh // 2
    case.pages.k[int(case.table[0, at // 16]), 0, at % 16, 3] = bad
    got = svod_amd.attention_paged(q, case.pages, Attn(causal=True))
    assert torch.equal(bits(got[:fresh // 2]), bits(want[:fresh // 2]))
    assert torch.isfinite(want).all()
    if bad != bad:
        assert torch.isnan(got[fresh // 2:]).all()
