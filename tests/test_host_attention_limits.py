"""Host side of the attention ops at the ends of their contract, no GPU."""
import ctypes

import pytest

import op_plugin_amd as q
from test_host_attention import _abi_cache

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
