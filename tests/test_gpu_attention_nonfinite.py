"""A seen infinity in V whose weight rounds to 0: the same answer in every tile, masked or not, and in either op."""
import math

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


@pytest.mark.parametrize("dtype,below", [(torch.float16, 60.0), (torch.bfloat16, 200.0)])
def test_infinity_without_weight(ops, dtype, below):
    """Key 0 has all the weight, key 10 e^-below of it, 0 in 16 bits: 0 times infinity, NaN, for every row that sees key 10."""
    print(f"[case] infinity without weight {dtype}", flush=True)
    g = torch.Generator().manual_seed(3)
    n, D = 400, 64
    q, k = torch.zeros((n, 2, D)), torch.zeros((n, 1, D))
    q[:, :, 0], k[0, 0, 0] = 1.0, below
    v = torch.randn((n, 1, D), generator=g)
    v[10, 0, 5], v[10, 0, 9] = math.inf, -math.inf
    q, k, v = (t.to(dtype).to(DEV) for t in (q, k, v))
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    out, _ = ops.npu_prompt_attention(q, k, v, cu, scale=1.0)
    bad = torch.zeros((n, 2, D), dtype=torch.bool)
    bad[10:, :, 5] = bad[10:, :, 9] = True
    assert torch.equal(torch.isnan(out).cpu(), bad) and torch.isfinite(out.cpu()[~bad]).all()
    table = torch.arange(n // 16, dtype=torch.int32, device=DEV)[None]
    for m in (11, 40, n):
        out, _ = ops.npu_paged_attention(q[:1], k.view(-1, 16, 1, D), v.view(-1, 16, 1, D), table,
                                         torch.tensor([m], dtype=torch.int32, device=DEV), scale=1.0)
        assert torch.equal(torch.isnan(out).cpu(), bad[-1:])
