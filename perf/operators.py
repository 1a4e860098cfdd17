"""A key/value cache kept in pages: written, read back and attended over, as cases that can be timed.

Four paths through three operators, each named after what calls it:

  write    the new tokens' keys and values go to their pages, 16 bits as they are (``write_pages``)
  store    the same into pages of 8 bits, quantised as they are written, and the sequences read back whole
           (``write_pages``, ``read_pages``): what a cache that is moved out and taken back costs
  read     the sequences of a cache read back in rows, for a call that wants them so (``read_pages``)
  attend   the attention of a step's new tokens over the pages of their sequences (``attention_paged``)

A cache is two pools ``[pages, kv_heads, page, head_dim]`` of 16-bit values, or of e4m3 codes with a power of two a row
(e8m0) as its scale.  Sequence b's token at position p lies in row ``p % page`` of page ``table[b, p // page]``; it has
``lens[b]`` tokens, of which the last ``starts[b + 1] - starts[b]`` are this step's, packed one sequence after the other.

The head counts are those of the models that the tests and the benchmark name; pages, batches and lengths are what a
serving loop sees, from one token of one sequence up.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# (query heads, KV heads, head size) of a layer's attention.
HEADS = {"qwen3": (16, 8, 128), "whisper": (20, 20, 64), "bge_m3": (16, 16, 64), "modernbert": (12, 12, 64)}
WIDE = (32, 8, 128)  # four query heads a KV head


def _case(name, path, batch, context, new, heads, page, dtype="bf16", cache="same", least=1.0, chunks=-1, causal=True,
          window=-1, tokens=0):
    """`batch` sequences of up to `context` earlier tokens, the shortest `least` of that; `chunks` of them (-1: all) bring
    `new` tokens each (down to `least` of that too), the others one.  `tokens`: rows a sequence that are read back (0: the
    longest's)."""
    h, hkv, d = heads
    c = {"path": path, "batch": batch, "context": context, "new": new, "least": least, "chunks": chunks, "heads": h,
         "kv_heads": hkv, "head_dim": d, "page": page, "dtype": dtype, "cache": cache, "causal": causal, "window": window,
         "tokens": tokens}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decoder step's keys and values into the cache, 16 sequences: the smallest call there is.  Latency.
        _case("write_step", "write", 16, 2100, 1, HEADS["qwen3"], 16, least=0.1),
        # A batch of prompts of odd lengths as they come out of the prologue, in f16.
        _case("write_prompts", "write", 8, 0, 2047, HEADS["whisper"], 32, "f16", least=0.2),
        # Prompts into a cache of 8 bits, and the sequences back in 16: the whole way there and back.
        _case("store_prompts", "store", 4, 0, 4096, HEADS["qwen3"], 16, cache="e4m3", least=0.5),
        # One token for each of a few short sequences in 8 bits: every launch is short.
        _case("store_step", "store", 5, 61, 1, HEADS["modernbert"], 16, "f16", "e4m3", least=0.3),
        # A long document's cache of 8 bits taken back into rows.
        _case("read_document", "read", 1, 32768, 0, HEADS["qwen3"], 64, cache="e4m3"),
        # A handful of prompts of odd lengths read back in 16 bits, fewer rows than the longest has.
        _case("read_prefix", "read", 7, 1201, 0, HEADS["bge_m3"], 32, "f16", least=0.2, tokens=777),
        # Generating: 16 sequences, a token each, over up to 2100 cached ones.
        _case("attend_step", "attend", 16, 2100, 1, HEADS["qwen3"], 16, least=0.1),
        # One sequence with a long document behind it: few rows, a long axis.
        _case("attend_document", "attend", 1, 65535, 1, HEADS["qwen3"], 64),
        # A full batch generating over a cache of 8 bits, four query heads a KV head.
        _case("attend_batch_e4m3", "attend", 64, 8192, 1, WIDE, 32, cache="e4m3", least=0.25),
        # Five drafted tokens a sequence to be checked at once, speech heads in f16.
        _case("attend_drafts", "attend", 9, 777, 5, HEADS["whisper"], 16, "f16", least=0.3),
        # A serving step: two prompts' chunks beside thirty sequences that generate, over 8 bits, in a window.
        _case("attend_mixed", "attend", 32, 1900, 1001, HEADS["qwen3"], 16, cache="e4m3", least=0.2, chunks=2, window=1024),
        # Chunks of long prompts: the largest call.
        _case("attend_chunks", "attend", 4, 16384, 2048, HEADS["qwen3"], 128, least=0.75),
    ]


def _spread(rng, low, high):
    """A whole number from `low` to `high`, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    path = rng.choice(["write", "store", "read"] + ["attend"] * 5)
    heads = rng.choice([*HEADS.values(), WIDE, (8, 1, 64), (15, 5, 128)])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = "e4m3" if path == "store" else "same" if path == "write" else rng.choice(["same", "e4m3"])
    least = round(rng.uniform(0.1, 1.0), 3)
    if path != "attend":
        rows = _spread(rng, 16, 16384)
        batch = _spread(rng, 1, max(1, min(64, rows)))
        each = max(1, rows // batch)
        if path == "read":
            return _case("", path, batch, each, 0, heads, page, dtype, cache, least, tokens=rng.choice([0, _spread(rng, 1, each)]))
        new = rng.choice([1, each])
        return _case("", path, batch, each - new, new, heads, page, dtype, cache, least)
    new = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 9, 2048)])
    context = rng.choice([0, _spread(rng, 1, 32768), _spread(rng, 1, 32768)])
    pairs = int(2e11 / (heads[0] * heads[2]))  # what one call may look at
    batch = _spread(rng, 1, max(1, min(64, pairs // (new * (context + new)), 200000 // (context + new))))
    chunks = rng.choice([-1, 1]) if new > 8 and batch > 1 else -1
    window = rng.choice([-1, -1, _spread(rng, 16, 4096)])
    return _case("", "attend", batch, context, new, heads, page, dtype, cache, least, chunks,
                 causal=window >= 0 or rng.random() < 0.85, window=window)


def _lengths(case):
    """(earlier tokens, new tokens) of each sequence: they go by the case alone, which sequence has which by the seed."""
    n, least = case["batch"], case["least"]
    share = [least + (1 - least) * (b + 1) / n for b in range(n)]
    chunks = n if case["chunks"] < 0 else min(case["chunks"], n)
    context = [int(round(case["context"] * s)) for s in share]
    new = [max(1, int(round(case["new"] * share[n - 1 - b]))) if b < chunks else 1 for b in range(n)]
    return [(c, t if case["new"] else 0) for c, t in zip(context, new)]


def _rows_back(case):
    return case["tokens"] or max(c + t for c, t in _lengths(case))


def _quantised(x):
    """Rows of e4m3 codes and their scales' exponents: 2^e is the least power of two with |row| <= 448 * 2^e.  Where a code
    would stand for more than the rows' own type holds, it is the largest that does not."""
    top = 8 if x.dtype == torch.float16 else 120
    x = x.float()
    amax = x.abs().amax(dim=-1)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -117)).clamp(min=-117)
    y = x * ((127 - e) << 23).view(torch.float32).unsqueeze(-1)
    limit = torch.where(e >= top, 240.0, 448.0).unsqueeze(-1)
    return torch.minimum(torch.maximum(y, -limit), limit).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)
    lengths = _lengths(case)
    random.Random(seed).shuffle(lengths)
    h, hkv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    lens = [c + t for c, t in lengths]
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device=device, dtype=torch.int64).to(torch.int32).tolist()
    table, at = torch.full((case["batch"], max(max(counts), 1)), -1, dtype=torch.int32), 0
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    starts = [0]
    for _, t in lengths:
        starts.append(starts[-1] + t)

    def rows(*shape):
        # A few channels of a head are much larger than the others, as keys have them.
        x = torch.randn(shape, generator=g, device=device)
        return (x * (1 + 3 * (torch.rand(shape[-1], generator=g, device=device) > 0.94))).to(dtype)

    new = starts[-1]
    state = {"case": case, "dtype": dtype, "tokens": _rows_back(case), "most_new": max(t for _, t in lengths),
             "table": table.to(device), "lens": torch.tensor(lens, dtype=torch.int32, device=device),
             "starts": torch.tensor(starts, dtype=torch.int32, device=device),
             "q": rows(new, h, d), "k": rows(new, hkv, d), "v": rows(new, hkv, d), "scales": (None, None)}
    pools = [rows(pages, hkv, page, d) for _ in range(2)]
    if case["cache"] == "e4m3":
        parts = [_quantised(x) for x in pools]
        pools = [codes for codes, _ in parts]
        state["scales"] = tuple(e.view(torch.float8_e8m0fnu) for _, e in parts)
    state["pools"] = tuple(pools)
    if own:
        import svod_amd
        from svod_amd import Attn, Pages

        state["pages"] = Pages(state["pools"][0], state["pools"][1], state["table"], state["lens"], state["starts"],
                               scales=None if state["scales"][0] is None else state["scales"])
        state["opts"] = Attn(causal=case["causal"], window=None if case["window"] < 0 else (case["window"], 0))
        state["ops"] = svod_amd
    return state


def _positions(state):
    """The sequence and the position of each new token."""
    starts, lens = state["starts"].long(), state["lens"].long()
    i = torch.arange(state["k"].shape[0], device=starts.device)
    b = torch.searchsorted(starts, i, right=True) - 1
    return b, lens[b] - starts[b + 1] + i


def _write(state):
    page = state["case"]["page"]
    b, at = _positions(state)
    to = state["table"].long()[b, at // page]
    for x, pool, scale in zip((state["k"], state["v"]), state["pools"], state["scales"]):
        if scale is None:
            pool[to, :, at % page] = x
        else:
            codes, e = _quantised(x)
            pool.view(torch.uint8)[to, :, at % page] = codes.view(torch.uint8)
            scale.view(torch.uint8)[to, :, at % page] = e


def _gathered(state, tokens):
    """Keys and values [batch, kv_heads, tokens, head_dim] in 32 bits, zeros past each sequence's end."""
    page, lens = state["case"]["page"], state["lens"].long()
    n = min(-(-tokens // page), state["table"].shape[1])
    at = state["table"].long()[:, :n].clamp(min=0)
    full = [x.view(torch.uint8)[at].view(x.dtype).float() if x.element_size() == 1 else x[at].float() for x in state["pools"]]
    if state["scales"][0] is not None:
        exponents = [s.view(torch.uint8)[at].int() for s in state["scales"]]
        full = [x * (e << 23).view(torch.float32).unsqueeze(-1) for x, e in zip(full, exponents)]
    inside = (torch.arange(tokens, device=lens.device) < lens[:, None])[:, None, :, None]
    # [batch, n, kv_heads, page, head_dim] -> [batch, kv_heads, n * page, head_dim]
    full = [x.transpose(1, 2).flatten(2, 3)[:, :, :tokens] for x in full]
    full = [torch.nn.functional.pad(x, (0, 0, 0, tokens - x.shape[2])) for x in full]
    return [torch.where(inside, x, torch.zeros((), device=x.device)) for x in full]


def _read(state):
    return tuple(x.transpose(1, 2).to(state["dtype"]).contiguous() for x in _gathered(state, state["tokens"]))


def _attend(state):
    case, q = state["case"], state["q"]
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    batch, most = case["batch"], state["most_new"]
    b, at = _positions(state)
    place = torch.arange(q.shape[0], device=q.device) - state["starts"].long()[b]
    padded = torch.zeros((batch, most, h, d), device=q.device)
    padded[b, place] = q.float()
    where = torch.zeros((batch, most), dtype=torch.int64, device=q.device)
    where[b, place] = at
    tokens = state["tokens"]
    k, v = _gathered(state, tokens)
    rows = padded.view(batch, most, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, d)
    scores = torch.matmul(rows, k.transpose(2, 3).contiguous()).view(batch, hkv, h // hkv, most, tokens)
    scores *= 1.0 / math.sqrt(d)
    key = torch.arange(tokens, device=q.device)
    seen = (key < state["lens"][:, None])[:, None, :]
    if case["causal"]:
        seen = seen & (key <= where[:, :, None])
    if case["window"] >= 0:
        seen = seen & (key >= where[:, :, None] - case["window"]) & (key <= where[:, :, None])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(dim=-1, keepdim=True)
    p = scores.exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(batch, hkv, -1, tokens), v).view(batch, hkv, h // hkv, most, d) / total
    return o.permute(0, 3, 1, 2, 4).reshape(batch, most, h, d)[b, place].to(q.dtype)


def run(state):
    path = state["case"]["path"]
    if own:
        ops, pages = state["ops"], state["pages"]
        if path == "write":
            ops.write_pages(state["k"], state["v"], pages)
            return state["pools"]
        if path == "store":
            ops.write_pages(state["k"], state["v"], pages)
            return ops.read_pages(pages, state["tokens"], state["dtype"])
        if path == "read":
            return ops.read_pages(pages, state["tokens"], state["dtype"])
        return ops.attention_paged(state["q"], pages, state["opts"])
    if path == "write":
        _write(state)
        return state["pools"]
    if path == "store":
        _write(state)
        return _read(state)
    if path == "read":
        return _read(state)
    return _attend(state)


def work(case):
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    lengths = _lengths(case)
    new = sum(t for _, t in lengths)
    row = hkv * (d + 1 if case["cache"] == "e4m3" else 2 * d)  # a token's keys (or values) in the cache
    wide = hkv * 2 * d
    ints = 4 * (2 * case["batch"] + 1)

    def table(tokens):
        return 4 * sum(-(-n // case["page"]) for n in tokens)

    rows = _rows_back(case)
    back = [min(c + t, rows) for c, t in lengths]
    taken_back = 2 * sum(back) * row + 2 * case["batch"] * rows * wide + table(back) + ints
    written = 2 * new * (wide + row) + 4 * new + ints
    if case["path"] == "write":
        return {"bytes": written, "flops": 0}
    if case["path"] == "store":
        return {"bytes": written + taken_back, "flops": 0}
    if case["path"] == "read":
        return {"bytes": taken_back, "flops": 0}
    pairs, keys = 0, []
    for c, t in lengths:
        left = case["window"] if case["window"] >= 0 else c + t
        if not case["causal"] and case["window"] < 0:
            pairs += t * (c + t)
        else:
            # The first tokens see all before them, those from position `left` on left + 1 keys.
            short = max(0, min(t, left - c))
            pairs += short * c + short * (short + 1) // 2 + (t - short) * (left + 1 if short < t else 0)
        keys.append(min(c + t, left + t))
    return {"bytes": 2 * sum(keys) * row + 2 * new * h * d * 2 + table(keys) + ints, "flops": 4 * pairs * h * d}


def exact(case, seed):
    """The definitions in 64 bits, a sequence at a time, on what `prepare` makes of the seed before anything has run."""
    state = prepare(case, seed)
    page, d, hkv = case["page"], case["head_dim"], case["kv_heads"]
    lens, starts = state["lens"].tolist(), state["starts"].tolist()
    table = state["table"].tolist()

    def power(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    def stored(x):
        """What a row is after it went into 8 bits and back: to four significant bits, 2^(e - 9) the least step."""
        x64 = x.double()
        amax = torch.clamp(x64.abs().amax(dim=-1, keepdim=True), min=2.0 ** -108)
        m, e = torch.frexp(amax / 448.0)
        e = torch.where(m == 0.5, e - 1, e)
        step = power(torch.clamp(torch.frexp(x64)[1] - 1 - e, min=-6) - 3 + e)
        y = torch.round(x64 / step) * step
        if x.dtype == torch.float16:
            most = 240.0 * power(e)
            y = torch.where(e >= 8, torch.minimum(torch.maximum(y, -most), most), y)
        return y

    def token_rows(which, b, n):
        """Sequence b's first n tokens [n, kv_heads, head_dim]."""
        pool, scale = state["pools"][which], state["scales"][which]
        ids = table[b][:-(-n // page)]
        parts = []
        for p in ids:
            x = pool[p].double()
            if scale is not None:
                x = x * power(scale[p].view(torch.uint8).int() - 127)[..., None]
            parts.append(x.transpose(0, 1))
        if not parts:
            return torch.zeros((0, hkv, d), dtype=torch.float64, device="cuda")
        return torch.cat(parts)[:n]

    if case["path"] == "write":
        pools = [x.double() for x in state["pools"]]
        for b, n in enumerate(lens):
            for i in range(starts[b], starts[b + 1]):
                at = n - (starts[b + 1] - i)
                for x, pool in zip((state["k"], state["v"]), pools):
                    pool[table[b][at // page], :, at % page] = x[i].double()
        return tuple(pools)
    if case["path"] in ("store", "read"):
        rows = state["tokens"]
        out = []
        for which, x in enumerate((state["k"], state["v"])):
            y = torch.zeros((case["batch"], rows, hkv, d), dtype=torch.float64, device="cuda")
            for b, n in enumerate(lens):
                whole = token_rows(which, b, n)
                if case["path"] == "store":
                    fresh = starts[b + 1] - starts[b]
                    whole = torch.cat([whole[:n - fresh], stored(x[starts[b]:starts[b + 1]])])
                y[b, :min(n, rows)] = whole[:rows]
            out.append(y)
        return tuple(out)
    q = state["q"].double()
    out = torch.zeros_like(q)
    for b, n in enumerate(lens):
        k, v = (token_rows(which, b, n) for which in (0, 1))
        s, e = starts[b], starts[b + 1]
        at = torch.arange(n - (e - s), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = torch.zeros((e - s, n), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= key > at
        if case["window"] >= 0:
            hidden |= (key < at - case["window"]) | (key > at)
        for head in range(case["heads"]):
            g = head * hkv // case["heads"]
            z = q[s:e, head] @ k[:, g].t() / math.sqrt(d)
            z = torch.softmax(z.masked_fill(hidden, -math.inf), dim=-1)
            out[s:e, head] = z @ v[:, g]
    return out
