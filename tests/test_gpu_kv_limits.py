"""npu_kv_extend where the pages and columns that are asked for pass what 16 or 32 bits count."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    return op_plugin_amd


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _refused(ops, table, lens, count, seqs, cu, total, missing):
    """`missing` is told, and nothing has changed."""
    slots, positions, got = ops.npu_kv_extend(table, lens, count, seqs, cu, total, 1)
    assert int(got) == missing
    assert (slots == -1).all() and (positions == -1).all()
    assert int(table.max()) == int(table.min()) == -1 and not lens.any() and not count.any()


@pytest.mark.parametrize("columns", [32768, 100000, 2 ** 31 - 11])
def test_missing_columns(ops, columns):
    print(f"[case] missing columns {columns}", flush=True)
    table, lens, count = torch.full((2, 10), -1, dtype=torch.int32, device=DEV), _ints([0, 0]), _ints([0] * 8)
    _refused(ops, table, lens, count, _ints([1]), _ints([0, columns + 10]), 3, columns)
    _refused(ops, table, lens, count, _ints([1, 0]), _ints([0, columns + 10, columns + 10]), 3, columns)


def test_missing_past_32_bits(ops):
    """2^32 pages and more between the sequences: sums that would come round to what the pool has."""
    print("[case] missing past 32 bits", flush=True)
    table, lens, count = torch.full((2, 10), -1, dtype=torch.int32, device=DEV), _ints([0, 0]), _ints([0] * 8)
    _refused(ops, table, lens, count, _ints([1]), _ints([-2 ** 31, 2 ** 31 - 1]), 3, 2 ** 31 - 1)
    n, width = 32768, 131073  # n * width = 2^32 + 32768
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    lens, count = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(40000, dtype=torch.int32, device=DEV)
    seqs = torch.full((2 * n,), -1, dtype=torch.int32, device=DEV)
    seqs[0::2] = torch.arange(n, dtype=torch.int32, device=DEV)
    cu = torch.zeros(2 * n + 1, dtype=torch.int32, device=DEV)
    cu[1::2] = width
    _refused(ops, table, lens, count, seqs, cu, 3, 2 ** 31 - 1)
