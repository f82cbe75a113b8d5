"""The attention ops at the ends of their contract: windows up to the largest number."""
import sys

import pytest
import torch

from test_gpu_attention import BF16, F16, _run_decode, _run_prompt, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,quant", [(0, False), (16, False), (16, True)])
@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31, 2 ** 40, sys.maxsize])
def test_prompt_window_without_end(ops, window, page, quant):  # noqa: F811
    """A window that holds every key is no window, also where a tile's first rows stand before the first key."""
    form = dict(k_lens=[70, 1, 0, 300], page=page, quant=quant)
    got = _run_prompt(ops, [140, 4, 2, 301], 2, 1, 64, window=window, sinks=3, **form)
    want = _run_prompt(ops, [140, 4, 2, 301], 2, 1, 64, **form)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("window", [2 ** 31 - 1, sys.maxsize])
def test_decode_window_without_end(ops, window):  # noqa: F811
    got = _run_decode(ops, [0, 1, 333], 4, 2, 64, 16, BF16, window=window, sinks=window)
    want = _run_decode(ops, [0, 1, 333], 4, 2, 64, 16, BF16)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("sinks", [2 ** 31 - 1, 2 ** 63 - 128, sys.maxsize])
def test_prompt_sinks_without_end(ops, sinks, quant):  # noqa: F811
    """With every key a sink a window hides nothing; few rows over a long past, so the keys are cut into parts."""
    got = _run_prompt(ops, [3, 1], 4, 1, 64, past=[3000, 700], page=16, quant=quant, window=100, sinks=sinks)
    want = _run_prompt(ops, [3, 1], 4, 1, 64, past=[3000, 700], page=16, quant=quant)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
