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


def test_many_wide_rows(ops):
    """Sums of 64 bits, over a batch that is padding but for three sequences, which get the lowest free pages in their order."""
    print("[case] many wide rows", flush=True)
    width, n = 40000, 65536
    table, lens = torch.full((3, width), -1, dtype=torch.int32, device=DEV), _ints([0, 0, 5])
    count = torch.zeros(width + 300, dtype=torch.int32, device=DEV)
    table[2, :2], count[[0, 7]] = _ints([7, 0]), 1
    seqs, grown = torch.full((n,), -1, dtype=torch.int32, device=DEV), torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    where = {10: (2, 6), 1500: (0, 9), 65535: (1, 4 * width)}
    for i, (seq, tokens) in where.items():
        seqs[i], grown[i + 1] = seq, tokens
    cu = grown.cumsum(0).to(torch.int32)
    total = int(cu[-1])
    slots, positions, missing = ops.npu_kv_extend(table, lens, count, seqs, cu, total, 4)
    assert int(missing) == 0 and lens.tolist() == [9, 4 * width, 11]
    free = [p for p in range(width + 300) if p not in (0, 7)]
    assert table[2, :4].tolist() == [7, 0, free[0], -1] and table[0, :4].tolist() == [*free[1:4], -1]
    assert table[1].tolist() == free[4:4 + width] and int(count.sum()) == 2 + 1 + 3 + width
    assert slots[:7].tolist() == [1, 2, 3, 4 * free[0], 4 * free[0] + 1, 4 * free[0] + 2, 4 * free[1]]
    assert positions[:7].tolist() == [5, 6, 7, 8, 9, 10, 0] and positions[15:].tolist() == list(range(4 * width))
    assert slots[-1] == 4 * free[3 + width] + 3
