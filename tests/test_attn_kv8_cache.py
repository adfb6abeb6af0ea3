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


@pytest.mark.parametrize("kv", [None, kv8.F8])
def test_append_kv_refuses_what_has_no_page(kv):
    """A call that would pass the capacity (48) raises before anything is stored."""
    c = _cache(kv_dtype=kv, scale_block=8)
    layer = c.cfg.attn_layers[0]
    x = torch.ones(2, c.cfg.num_key_value_heads, 20, c.cfg.head_dim)
    c.append_kv(layer, x, x)
    c.append_kv(layer, x, x)
    before = c.k_pages.view(torch.uint8).clone()
    with pytest.raises(RuntimeError, match="capacity"):
        c.append_kv(layer, 2 * x, x)
    assert torch.equal(c.k_pages.view(torch.uint8), before) and c.seen_tokens == 40
