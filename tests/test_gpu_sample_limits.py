"""npu_sample where rows leave the usual paths: borders among thousands of near tokens, vocabularies past what a split row holds, as
many rows as a launch takes."""
import pytest
import torch

from test_gpu_sample import BF16, DEV, F16, F32, _check, _logits, _settings, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [6, 200])
@pytest.mark.parametrize("scale", [0.03, 0.1, 0.2, 0.4])
def test_borders_among_near_tokens(ops, scale, R):  # noqa: F811
    """From some hundreds to more tokens in the border's bins than are listed."""
    g = torch.Generator().manual_seed(int(100 * scale) + R)
    V = 40000
    for dtype in (F32, F16):
        x = _logits(g, R, V, dtype, scale=scale, peaks=0)
        u = torch.rand(R, generator=g)
        _check(ops, x, u, k=torch.randint(1, V, (R,), generator=g))
        _check(ops, x, u, p=0.05 + 0.9 * torch.rand(R, generator=g))
        _check(ops, x, u, k=torch.randint(V // 4, V, (R,), generator=g), p=0.3 + 0.7 * torch.rand(R, generator=g))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [(1 << 20) - 8, (1 << 20) - 7, (1 << 20) + 5, 1300001])
def test_large_vocabularies(ops, V, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(V)
    x, u = _logits(g, 4, V, dtype), torch.rand(4, generator=g)
    _check(ops, x, u)
    _check(ops, x, u, t=torch.tensor([0.0, 0.5, 1.0, 2.0]), k=torch.tensor([0, 5, 700, 0]), p=torch.tensor([1.0, 0.9, 0.999, 0.95]),
           m=torch.tensor([0.0, 0.0, 0.01, 0.1]))


def test_as_many_rows_as_a_launch_takes(ops):  # noqa: F811
    """Two equal logits: the second from a half on."""
    R = (1 << 22) - 1
    print(f"[case] sample {R} x 2", flush=True)
    u = torch.rand(R, generator=torch.Generator().manual_seed(1)).to(DEV)
    tokens, _ = ops.npu_sample(torch.zeros((R, 2), dtype=BF16, device=DEV), u)
    assert torch.equal(tokens, (u >= 0.5).to(torch.int32))
