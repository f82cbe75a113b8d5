"""One key with nearly all the weight over 131071 with some 2^-25.5 each: together they carry what float16 would show, and no
weight of them is a normal number of that type beside the largest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16
N, D, PAGE = 131072, 64, 128


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import op_plugin_amd
    return op_plugin_amd


def _caches(dtype, quant):
    """The cache in order of its tokens, its scales, and the scores and values that it means, in 64 bits; q = e_0, scale 1."""
    g = torch.Generator().manual_seed(1)
    below = (25.1 + 0.9 * torch.rand(N, generator=g)) * math.log(2)  # scores under the first key's
    below[0] = 0.0
    k, v = torch.zeros((N, 1, D)), torch.randint(64, 128, (N, 1, D), generator=g).float()
    v[0] = 0.0
    if quant:
        k[:, 0, 0] = -127.0 * (below > 0)
        ks, vs = below[:, None] / 127, torch.full((N, 1), 1 / 127)
        kc, vc = k.to(torch.int8), v.to(torch.int8)
        s, vv = kc[:, 0, 0].double() * ks[:, 0].double(), vc[:, 0].double() * vs.double()
        ks, vs = ks.view(-1, PAGE, 1).to(DEV), vs.view(-1, PAGE, 1).to(DEV)
    else:
        k[:, 0, 0], v = -below, v / 127
        kc, vc, ks, vs = k.to(dtype), v.to(dtype), None, None
        s, vv = kc[:, 0, 0].double(), vc[:, 0].double()
    return kc.view(-1, PAGE, 1, D).to(DEV), vc.view(-1, PAGE, 1, D).to(DEV), ks, vs, s, vv


def _check(out, lse, s, v, dtype):
    """A weight is off by half a step u, relative, where it is at least 2^-21 of the row's largest, else by 2^-32 of that; the
    result by half a step. In 32 bits: scores of one product, exponentials, and sums of N weights."""
    w = torch.exp(s - s.max())
    total = w.sum()
    want, size = (w @ v) / total, (w @ v.abs()) / total
    u, f = torch.finfo(dtype).eps / 2, 2.0 ** -24
    delta = (float(s.abs().max()) * (D + 8) + N + 64) * f
    tol = size * (u + 2 * delta) * (1 + 2 * u) + want.abs() * u + N * 2.0 ** -32 * v.abs().max() / total + 2.0 ** -25
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(out, out[:1].expand_as(out)), "every sequence is the same"
    worst = float(((out[0] - want).abs() / tol).max())
    assert worst <= 1, f"{worst:.2f} of the bound"
    assert ((lse - (s.max() + total.log())).abs() <= delta).all()


@pytest.mark.parametrize("dtype,quant", [(F16, False), (F16, True), (BF16, True), (BF16, False)])
@pytest.mark.parametrize("phase", ["decode", "prompt"])
def test_small_weights_add_up(ops, phase, dtype, quant):
    """So many sequences, all of the same pages, that the keys of none are cut."""
    print(f"[case] tail {phase} {dtype} quant={quant}", flush=True)
    kc, vc, ks, vs, s, v = _caches(dtype, quant)
    B = 768 if phase == "decode" else 512
    q = torch.zeros((B, 1, D), dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    table = torch.arange(N // PAGE, dtype=torch.int32, device=DEV).expand(B, -1)
    lens = torch.full((B,), N, dtype=torch.int32, device=DEV)
    if phase == "decode":
        out, lse = ops.npu_paged_attention(q, kc, vc, table, lens, key_scale=ks, value_scale=vs, scale=1.0)
    else:
        out, lse = ops.npu_prompt_attention(q, kc, vc, torch.arange(B + 1, dtype=torch.int32, device=DEV), block_table=table,
                                            context_lens=lens, key_scale=ks, value_scale=vs, scale=1.0)
    _check(out[:, 0], lse[:, 0], s, v, dtype)
