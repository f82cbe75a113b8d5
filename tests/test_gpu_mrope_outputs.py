"""qk_mrope with an output that the caller does not want (NULL): the others as with both."""
import ctypes

import pytest
import torch

import op_plugin_amd as q

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D,rot", [(64, 64), (72, 40)])  # the kernel of whole pieces, and the one for any form
@pytest.mark.parametrize("cached", [False, True])
@pytest.mark.parametrize("want_q,want_k", [(True, True), (True, False), (False, True), (False, False)])
def test_null_outputs(want_q, want_k, cached, D, rot):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    print(f"[case] null outputs D={D} cached={cached} {want_q} {want_k}", flush=True)
    g = torch.Generator().manual_seed(1)
    T, Hq, Hkv, page = 5, 3, 2, 4
    x, k, v = (torch.randn((T, h, D), generator=g).to(torch.bfloat16).to(DEV) for h in (Hq, Hkv, Hkv))
    table = torch.randn((50, rot), generator=g).to(DEV)
    positions = torch.randint(0, 50, (T,), generator=g, dtype=torch.int32).to(DEV)
    slots = torch.tensor([3, -1, 0, 9, 5], dtype=torch.int32, device=DEV)
    turned_q, turned_k = q.npu_mrope(positions, x, k, table)
    out_q, out_k = torch.full_like(x, 7.0), torch.full_like(k, 7.0)
    kc, vc = (torch.full((3, page, Hkv, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cache = q.KvCache(key=kc.data_ptr(), value=vc.data_ptr(), num_pages=3, page_size=page, kv_heads=Hkv, head_dim=D,
                      key_page_stride=kc.stride(0), key_token_stride=kc.stride(1), key_head_stride=kc.stride(2),
                      value_page_stride=vc.stride(0), value_token_stride=vc.stride(1), value_head_stride=vc.stride(2),
                      dtype=q.QK_BF16)
    rc = q.abi().qk_mrope(x.data_ptr(), k.data_ptr(), v.data_ptr() if cached else None, q.QK_BF16, T, Hq, Hkv, D, Hq * D, D,
                          Hkv * D, D, Hkv * D, D, positions.data_ptr(), 1, 0, None, table.data_ptr(), q.QK_F32, 50, rot, 0,
                          out_q.data_ptr() if want_q else None, out_k.data_ptr() if want_k else None,
                          ctypes.byref(cache) if cached else None, slots.data_ptr() if cached else None,
                          ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == q.QK_OK, q.last_error()
    seven = lambda t: torch.full_like(t, 7.0)  # noqa: E731
    assert torch.equal(out_q, turned_q if want_q else seven(out_q)) and torch.equal(out_k, turned_k if want_k else seven(out_k))
    put = slots >= 0
    for rows, out in ((turned_k, kc), (v, vc)):
        want = seven(out).flatten(0, 1)
        if cached:
            want[slots[put].long()] = rows[put]
        assert torch.equal(out.flatten(0, 1), want)
