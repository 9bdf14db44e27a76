"""The workspace of attention over an 8-bit cache: what it allocates, and that the memory plan counts it."""

import pytest
import torch

from eagle4_b200.api import NAMED
from eagle4_b200.ops.quant import attention_workspace, kv_code, new_cache
from eagle4_b200.runtime.memory import plan


@pytest.mark.parametrize("tp", [1, 4])
def test_the_memory_plan_counts_the_attention_workspace(tp):
    tcfg = NAMED["qwen3.8-27b"][0]()
    dcfg = NAMED["qwen3.8-27b"][1](tcfg)
    kw = dict(tp=tp, max_batch=4, max_len=65536, tree=(12, 4, 16))
    p16, p8 = (plan(tcfg, dcfg, kv_dtype=k, **kw) for k in (None, "int8"))
    hq, hk = (tcfg.num_heads, tcfg.num_kv_heads) if tp == 1 else (tcfg.num_heads // tp, max(1, tcfg.num_kv_heads // tp))
    row = 65536 + 12 * 4 + 1
    want = sum(attention_workspace(t, hq, hk, tcfg.head_dim, row) for t in (8192, 4 * 16))
    assert p16.attention == 0 and p8.attention == want > 0
    assert p8.total == p8.weights + p8.kv + p8.state_bytes + p8.reserve + p8.prefill + want
    budget = p8.total
    assert budget - p8.kv + p8.kv_tokens_within(budget) * p8.kv_bytes_per_token <= budget
    assert p8.summary(100.0)["attention"] == round(want / 1e9, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hq,hk,d,max_keys", [
    (1, 24, 4, 256, 4096), (32, 6, 1, 256, 32768), (300, 4, 1, 128, 65536), (32, 16, 1, 256, 32768), (5, 64, 8, 128, 1000),
    (1, 4, 4, 64, 10), (1, 1, 1, 16, 1)])
def test_what_a_call_allocates(rows, hq, hk, d, max_keys):
    from eagle4_b200 import ops

    kc, vc = (new_cache(64, hk, d, torch.bfloat16, kv_code("fp8"), "cuda") for _ in range(2))
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (torch.zeros(rows, hq, d, dtype=torch.bfloat16, device="cuda"), kc, vc, i32(1, 4), 16, i32(rows), i32(rows),
            i32(rows), i32(rows, 1), i32(rows), 0.1, max_keys)
    ops.attention(*args)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.attention(*args)
    grown = torch.cuda.max_memory_allocated() - before - -(-out.numel() * 2 // 512) * 512
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    want = attention_workspace(rows, hq, hk, d, max_keys, sms)
    assert want <= grown <= want + 1024  # (the allocator's rounding)
