"""PagedKVCache's own state on the host, no GPU."""
import torch

from op_plugin_amd.kv_cache import PagedKVCache


def _ints(v):
    return torch.tensor(v, dtype=torch.int32)


def test_rows_of_padding():
    """A batch's padding has no tokens, whatever the last sequence holds."""
    cache = PagedKVCache(1, 8, 4, 1, 16, max_seqs=3, max_len=8, device="cpu")
    cache.block_table[2], cache.block_table[0] = _ints([5, 6]), _ints([1, -1])
    cache.context_lens[2], cache.context_lens[0] = 7, 2
    table, lens = cache.rows(_ints([0, -1, 2, 3, 2 ** 31 - 1, -2 ** 31, 1]))
    assert lens.tolist() == [2, 0, 7, 0, 0, 0, 0] and lens.dtype == table.dtype == torch.int32
    assert table[0].tolist() == [1, -1] and table[2].tolist() == [5, 6] and table[6].tolist() == [-1, -1]
    table, lens = PagedKVCache(1, 8, 4, 1, 16, max_seqs=0, max_len=8, device="cpu").rows(_ints([0, -1]))
    assert lens.tolist() == [0, 0] and table.tolist() == [[-1, -1]] * 2


def test_scales_are_float32():
    """... whatever torch's default is: the ops take no other."""
    before = torch.get_default_dtype()
    try:
        for default in (torch.float64, torch.bfloat16):
            torch.set_default_dtype(default)
            cache = PagedKVCache(2, 8, 4, 3, 16, max_seqs=2, max_len=8, dtype=torch.int8, device="cpu")
            for s in cache.key_scales + cache.value_scales:
                assert s.dtype == torch.float32 and s.shape == (8, 4, 3)
    finally:
        torch.set_default_dtype(before)
