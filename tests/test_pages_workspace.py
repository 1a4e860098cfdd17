"""The workspace of attention over pages without a GPU: partial states for the workgroups that a launch has."""
import pytest
import torch

import svod_amd
from svod_amd import Attn, Pages


@pytest.mark.parametrize("kv_heads", [1, 3, 5, 7, 8])
@pytest.mark.parametrize("coded", [False, True])
def test_shares_have_states_for_the_workgroups_that_are_launched(kv_heads, coded):
    """One token each of many sequences, whose blocks may be shared out over the chip's places: three workgroups of tiles of 16 rows of 64
    on each of 256 units, in whole rounds of the KV heads, each with two states; and a line of memory for every workgroup."""
    batch, d, page = 400, 64, 16
    dtype = torch.float8_e4m3fn if coded else torch.bfloat16
    pool = lambda: torch.zeros(4, kv_heads, page, d, dtype=torch.uint8 if coded else dtype).view(dtype)
    scale = lambda: torch.zeros(4, kv_heads, page, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    pages = Pages(pool(), pool(), torch.zeros(batch, 200, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32),
                  torch.zeros(batch + 1, dtype=torch.int32), (scale(), scale()) if coded else None)
    q = torch.zeros(batch, 2 * kv_heads, d, dtype=torch.bfloat16)
    on_places = (256 * 3 // kv_heads + 1) * kv_heads
    workgroups = max(batch * kv_heads, on_places)
    state = 16 * (d + 2) * 4
    assert svod_amd.attention_paged_workspace(q, pages, Attn(causal=True)) == 2 * on_places * state + workgroups * 128


def test_a_chunk_over_few_keys_is_not_split():
    """Below eight key blocks a tile of 128 rows stays whole whatever the lengths, so that no merge is launched."""
    def bytes_of(keys, d=128):
        pool = lambda: torch.zeros(4, 8, 64, d, dtype=torch.bfloat16)
        pages = Pages(pool(), pool(), torch.zeros(1, keys // 64, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                      torch.zeros(2, dtype=torch.int32))
        return svod_amd.attention_paged_workspace(torch.zeros(128, 16, d, dtype=torch.bfloat16), pages, Attn(causal=True))

    for d in (64, 128, 256):
        assert [bytes_of(64 * n, d) > 0 for n in (1, 4, 5, 7, 8, 9)] == [False] * 4 + [True] * 2
