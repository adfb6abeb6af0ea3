"""The family cache, on the CPU: what it refuses."""

import pytest
import torch

from oracle import kv8


def _cache(raw=None, ps=16, **kw):
    from lollm_b200.qwen3_5 import Qwen3_5Cache, Qwen3_5Config
    from lollm_b200.qwen3_5.config import MICRO
    return Qwen3_5Cache(Qwen3_5Config.from_hf(raw or MICRO), 2, 40, dtype=torch.bfloat16, device="cpu", page_size=ps, **kw)


@pytest.mark.parametrize("kw", [dict(head_dim=48), dict(head_dim=512), dict(head_dim=256, partial_rotary_factor=0.28125)])
def test_cache_refuses_heads_that_no_kernel_takes(kw):
    """Where the cache is made, not at the first forward; a 16-bit cache of the same heads is made."""
    from lollm_b200.qwen3_5.config import MICRO
    raw = dict(MICRO, text_config=dict(MICRO["text_config"], **kw))
    with pytest.raises(RuntimeError, match="8-bit"):
        _cache(raw, kv_dtype=kv8.F8)
    _cache(raw)
