"""The ops over a key/value cache in pages without a GPU: what they refuse, and what they leave to the graph."""
import pytest
import torch

import svod_amd
from svod_amd import Attn, GraphFallback, KeyMask, OpError, Pages

BF16, F16, F32, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype) if dtype in (E4M3, E8M0) else torch.zeros(shape, dtype=dtype)


def pages(coded=False, **changed):
    fields = dict(k=t(6, 2, 16, 64, dtype=E4M3 if coded else BF16), v=t(6, 2, 16, 64, dtype=E4M3 if coded else BF16),
                  table=t(3, 4, dtype=I32), lens=t(3, dtype=I32), starts=t(4, dtype=I64),
                  scales=(t(6, 2, 16, dtype=E8M0), t(6, 2, 16, dtype=E8M0)) if coded else None)
    return Pages(**{**fields, **changed})


Q, KV = t(5, 4, 64), t(5, 2, 64)
attend = lambda p=None, q=Q, opts=None, **kw: svod_amd.attention_paged(q, p or pages(), opts, **kw)
write = lambda p=None, k=KV, v=KV: svod_amd.write_pages(k, v, p or pages())
read = lambda p=None, tokens=7, **kw: svod_amd.read_pages(p or pages(), tokens, **kw)


@pytest.mark.parametrize("call,kind", [
    (lambda: attend(pages(k=t(6, 2, 16))), "Shape"),
    (lambda: attend(pages(v=t(6, 2, 32, 64))), "Shape"),
    (lambda: attend(pages(v=t(6, 2, 16, 64, dtype=F16))), "Dtype"),
    (lambda: attend(pages(table=t(3, dtype=I32))), "Shape"),
    (lambda: attend(pages(table=t(3, 4, dtype=I64))), "Dtype"),
    (lambda: attend(pages(lens=t(4, dtype=I32))), "Shape"),
    (lambda: attend(pages(lens=t(3, dtype=F32))), "Dtype"),
    (lambda: attend(pages(starts=t(3, dtype=I32))), "Shape"),
    (lambda: attend(pages(starts=t(4, dtype=BF16))), "Dtype"),
    (lambda: attend(pages(starts=None)), "Argument"),
    (lambda: write(pages(starts=None)), "Argument"),
    (lambda: attend(pages(scales=(t(6, 2, 16, dtype=E8M0),) * 2)), "Argument"),
    (lambda: attend(pages(coded=True, scales=None)), "Argument"),
    (lambda: attend(pages(coded=True, scales=(t(6, 2, 16, dtype=E8M0), t(6, 2, 8, dtype=E8M0)))), "Shape"),
    (lambda: attend(pages(coded=True, scales=(t(6, 2, 16), t(6, 2, 16)))), "Dtype"),
    (lambda: attend(q=t(5, 4, 128)), "Shape"),
    (lambda: attend(q=t(1, 5, 4, 64)), "Shape"),
    (lambda: attend(q=t(5, 3, 64)), "Heads"),
    (lambda: attend(q=t(5, 0, 64)), "Heads"),
    (lambda: attend(q=t(5, 4, 64, dtype=F16)), "Dtype"),
    (lambda: attend(out=t(5, 2, 64)), "Shape"),
    (lambda: attend(out=t(5, 4, 64, dtype=F16)), "Dtype"),
    (lambda: attend(opts=Attn(window=(-1, 0))), "Argument"),
    (lambda: attend(q=t(4, 5, 64).transpose(0, 1)), "Argument"),
    (lambda: write(k=t(5, 3, 64), v=t(5, 3, 64)), "Shape"),
    (lambda: write(k=t(5, 2, 128), v=t(5, 2, 128)), "Shape"),
    (lambda: write(v=t(4, 2, 64)), "Shape"),
    (lambda: write(v=t(5, 2, 64, dtype=F16)), "Dtype"),
    (lambda: write(k=t(5, 2, 64, dtype=F16), v=t(5, 2, 64, dtype=F16)), "Dtype"),
    (lambda: read(out=(t(3, 7, 2, 64), t(3, 8, 2, 64))), "Shape"),
    (lambda: read(out=(t(2, 7, 2, 64), t(2, 7, 2, 64))), "Shape"),
    (lambda: read(out=(t(3, 7, 2, 64), t(3, 7, 2, 64, dtype=F16))), "Dtype"),
    (lambda: read(dtype=F16), "Dtype"),
    (lambda: read(dtype=torch.float64), "Dtype"),
    (lambda: read(tokens=-1), "Shape"),
])
def test_refused(call, kind):
    with pytest.raises(OpError) as e:
        call()
    assert e.value.kind == kind, e.value


def test_what_is_no_dtype_is_a_type_error():
    with pytest.raises(TypeError):
        read(dtype=3)


@pytest.mark.parametrize("call", [attend, write, read, lambda: attend(pages(coded=True)), lambda: write(pages(coded=True)),
                                  lambda: read(pages(coded=True), dtype=F16)])
def test_without_a_device_the_graph_runs(call):
    if torch.cuda.is_available():
        pytest.skip("a device is here")
    with pytest.raises(GraphFallback) as e:
        call()
    assert e.value.why == svod_amd.Fallback.Target


def test_the_workspace_follows_the_form():
    w = svod_amd.attention_paged_workspace
    short, long = pages(table=t(3, 4, dtype=I32)), pages(table=t(3, 400, dtype=I32))
    state = lambda rows: rows * 66 * 4
    assert w(Q, short, Attn(causal=True)) == 0  # one key block at most: never split
    assert w(Q, long, Attn(causal=True, splits=1)) == 0
    # Five rows of two heads a KV head in three sequences: 16 rows a tile, a state and a line of memory for each place of the chip
    # (the six tiles there may be are fewer).
    few = w(Q, long, Attn(causal=True))
    assert few > 0 and few % (state(16) + 128) == 0
    many = w(t(900, 4, 64), long, Attn(causal=True))  # 128 rows a tile
    assert many > 0 and (many - 16) % state(128) == 0
    # A named count: that many states for each tile, three a KV head.
    assert w(Q, long, Attn(causal=True, splits=7)) == 3 * 2 * 7 * (state(16) + 128)
    assert w(Q, short, Attn(causal=True, splits=7)) == 0  # no more splits than key blocks: one
    # What the op would not take asks for nothing.
    assert w(t(5, 3, 64), long, Attn()) == 0 and w(Q, long, Attn(keys=KeyMask.lens(t(3, dtype=I32)))) == 0
