"""What is more than a launch can have is refused by name, before anything is launched."""
import ctypes

import pytest

from test_paged_cache import CACHE, STEP
from test_paged_conversations import EVICTION, STEPS


@pytest.mark.parametrize("batch,heads", [(65535, 65), (65536 // 2, 128), (1 << 15, 255)])
def test_evictions_of_too_many_sequences_and_heads(batch, heads):
    """2^22 work-groups of 1024 threads are 2^32."""
    from anchor_attn.src.ops import _hip
    struct = _hip.PagedCacheStruct(*{**CACHE, "n_kv_heads": heads, "kp_sh": 128}.values())
    with pytest.raises(_hip.AnchorAttnHipError, match="fewer than 2\\^22"):
        _hip.check(_hip.lib().aa_paged_evict(ctypes.addressof(struct), _hip.PAGED_EVICTION.pack(*{**EVICTION, "batch": batch}.values()), None))


@pytest.mark.parametrize("fn,batch,heads,message", [
    ("weigh", 65535, 256, "2\\^24 - 4096"), ("weigh", 4097, 4095, "2\\^24 - 4096"), ("shared", 4097, 4095, "2\\^24 - 8"), *[(fn, 4096, 4096, "2\\^24") for fn in STEPS],
])
def test_steps_of_too_many_sequences_and_heads(fn, batch, heads, message):
    from anchor_attn.src.ops import _hip
    name, more = STEPS[fn]
    struct = _hip.PagedCacheStruct(*{**CACHE, "n_kv_heads": heads}.values())
    step = _hip.PAGED_STEP.pack(*{**STEP, "batch": batch, "n_q_heads": heads, "max_pages": 1}.values())
    with pytest.raises(_hip.AnchorAttnHipError, match=message):
        _hip.check(getattr(_hip.lib(), name)(ctypes.addressof(struct), step, *more.values(), None))
