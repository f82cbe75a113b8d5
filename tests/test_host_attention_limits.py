"""Host side of the attention ops at the ends of their contract, no GPU."""
import ctypes
import math

import pytest

import op_plugin_amd as q
from test_host_attention import I32, _abi_cache, _cache, _m

LAST = 2 ** 63 - 1


@pytest.mark.parametrize("window", [1, 100, 4096, 2 ** 31, LAST])
@pytest.mark.parametrize("sinks", [2 ** 31, LAST - 128, LAST - 127, LAST])
def test_workspace_of_sinks_without_end(window, sinks):
    """The workspace query takes a number past 31 bits as the launch does: as 2^31 - 1."""
    L, c = q.abi(), _abi_cache(num_pages=4000)
    most = 2 ** 31 - 1

    def sizes(w, s):
        a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
        assert L.qk_prompt_attention_workspace_size(4, 1, 8, ctypes.byref(c), 2000, w, s, ctypes.byref(a)) == q.QK_OK
        assert L.qk_paged_attention_workspace_size(4, 8, ctypes.byref(c), 2000, w, s, ctypes.byref(b)) == q.QK_OK
        return a.value, b.value

    assert sizes(window, sinks) == sizes(min(window, most), most)
    assert sizes(window, sinks)[0] > 0  # 32000 keys under four tokens are cut into parts


@pytest.mark.parametrize("scale", [1e300, -1e300, 3.5e38, 3e38, -2.4e38, math.inf, math.nan])
def test_scales_that_float32_cannot_hold(scale):
    """... times log2 e, which the kernels multiply scores by: refused by the ops and by the C ABI."""
    k, v = _cache()
    with pytest.raises(RuntimeError, match="scale must be finite"):
        q.npu_paged_attention(_m((3, 8, 64)), k, v, _m((3, 5), I32), _m((3,), I32), scale=scale)
    with pytest.raises(RuntimeError, match="scale must be finite"):
        q.npu_prompt_attention(_m((30, 8, 64)), _m((30, 2, 64)), _m((30, 2, 64)), _m((4,), I32), scale=scale)
    L, fake, c = q.abi(), ctypes.c_void_p(4096), ctypes.byref(_abi_cache(num_pages=1))
    at = ctypes.c_float(scale)
    assert L.qk_paged_attention(fake, q.QK_BF16, 3, 8, 512, 64, c, fake, 5, 5, fake, at, 0, 0, fake, fake, None, 0,
                                None) == q.QK_ERR_ARG and "scale" in q.last_error()
    assert L.qk_prompt_attention(fake, q.QK_BF16, 9, 3, 8, 512, 64, fake, c, fake, None, 0, 0, None, at, 0, 0, fake, None, None,
                                 0, None) == q.QK_ERR_ARG and "scale" in q.last_error()


@pytest.mark.parametrize("scale", [2.3e38, -2.3e38, 1e-300, 0.0, -0.5])
def test_scales_that_it_can(scale):
    k, v = _cache()
    q.npu_paged_attention(_m((3, 8, 64)), k, v, _m((3, 5), I32), _m((3,), I32), scale=scale)
    q.npu_prompt_attention(_m((30, 8, 64)), _m((30, 2, 64)), _m((30, 2, 64)), _m((4,), I32), scale=scale)


@pytest.mark.parametrize("n", [0, 1, 2, 1000])
def test_fork_workspace(n):
    """A byte less than the query says is refused (checked before any launch)."""
    L, fake, size = q.abi(), ctypes.c_void_p(4096), ctypes.c_size_t(0)
    assert L.qk_kv_fork_workspace_size(n, ctypes.byref(size)) == q.QK_OK
    assert size.value == 4 * (3 * n + 1)  # sources, destinations, the new pages, and whether there are enough
    assert L.qk_kv_fork(None, 0, 5, 16, fake, 4, 8, 8, fake, fake, fake, fake, n, fake, fake, size.value - 1,
                        None) == q.QK_ERR_WORKSPACE and str(size.value) in q.last_error()
