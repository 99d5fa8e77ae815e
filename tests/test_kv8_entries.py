"""What the 8-bit cache refuses without a GPU, beyond shapes, types and pointers of one call."""
import math

import pytest
import torch


@pytest.mark.parametrize("scale", [0.0, -0.125, math.nan, math.inf, -math.inf, 3.0e38])
@pytest.mark.parametrize("window", [False, True])
def test_prompt_attention_refuses_factors_it_cannot_mask_with(scale, window):
    """The kernel takes the maximum of the scores before their factor, and -inf times 0 is NaN."""
    from acorninfer_amd import _lib
    p = 64                                              # a pointer that is never followed
    meta = None if window else p
    assert _lib.lib().acorn_paged_prefill_attention_kv8(
        p, p, p, p, p, meta, p, meta, p, 1, 1, 1, 2, 2, 64, 16, 4, 1, scale, 2, None, 0,
        None) == _lib.ERR_VALUE


@pytest.mark.parametrize("layers,KV,D", [(1, 8, 128), (2, 4, 128), (2, 16, 128), (2, 8, 64)])
def test_a_cache_of_another_models_shape_is_refused(layers, KV, D):
    """A step reaches the pools by the model's own layers, kv heads and head_dim."""
    from types import SimpleNamespace

    from acorninfer_amd.cache.pager import BlockAllocator, PagedKV8Cache
    from acorninfer_amd.config import Qwen3Config
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel
    cfg = Qwen3Config.qwen3_0_6b().with_layers(2)
    assert (cfg.num_key_value_heads, cfg.head_dim) == (8, 128)
    w = torch.ones(128, dtype=torch.bfloat16)
    model = SimpleNamespace(cfg=cfg, dtype=torch.bfloat16,
                            layers=[SimpleNamespace(q_norm=w, k_norm=w) for _ in range(2)])
    for n in (2, 3):                                    # (layers that no step reads do no harm)
        good = PagedKV8Cache(n, 8, 128, 16, BlockAllocator(2), "cpu", torch.bfloat16)
        assert Qwen3DecodeModel.kv8_page(model, good) == 16
    with pytest.raises(ValueError):
        Qwen3DecodeModel.kv8_page(model, PagedKV8Cache(layers, KV, D, 16, BlockAllocator(2), "cpu",
                                                       torch.bfloat16))
