"""Tensor-parallel ranks over an 8-bit KV cache (gloo on the CPU), and attention over one on two streams."""

import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(1)
    try:
        from eagle4_b200.api import LLM, TreeSpec
        from eagle4_b200.models.target import RowBatch
        from eagle4_b200.parallel.tp import TensorParallel

        kw = dict(device="cpu", dtype=torch.float32, tree=TreeSpec(4, 2, 8), max_len=128, kv_dtype="int8")
        llm, ref = LLM.synthetic("tiny", tp=TensorParallel(backend="torch"), **kw), LLM.synthetic("tiny", **kw)
        prompt = torch.randint(0, 4096, (24,), generator=torch.Generator().manual_seed(0))
        n, pos = 24, torch.arange(24)
        rows = []
        for m in (llm, ref):
            eng = m.engine
            eng.pages.reserve(0, n + 1)
            slots = eng._slots(torch.tensor(0), pos)
            i32 = torch.zeros(n, dtype=torch.int32)
            rb = RowBatch(ids=prompt, pos=pos, req=i32, write_slot=slots, ctx_start=i32, ctx_len=(pos + 1).int(),
                          extra=i32[:, None], n_extra=i32, parent=(pos - 1).int(), state_slot=i32, scan=True)
            m.target.forward(rb, eng.tcache)
            rows.append([(c.data[slots].int(), c.scale[:, slots]) for c in (eng.tcache.k[0], eng.tcache.v[0])])
        codes = scales = 0
        for (mine, s), (whole, t) in zip(*rows):
            codes = max(codes, (mine[:, 0] - whole[:, rank]).abs().max().item())
            scales = max(scales, ((s[0] - t[rank]) / t[rank]).abs().max().item())
        spec, plain = llm.generate(prompt[None], 12), llm.generate(prompt[None], 12, speculative=False)
        gathered = [None] * world
        dist.all_gather_object(gathered, spec.tolist())
        out[rank] = {"heads": llm.engine.tcache.k[0].shape[1], "codes": codes, "scales": scales,
                     "spec_eq_plain": bool(torch.equal(spec, plain)), "ranks_agree": all(x == gathered[0] for x in gathered)}
    finally:
        dist.destroy_process_group()


def test_ranks_hold_their_heads_of_the_8_bit_cache():
    """Each rank's codes are the single process's codes of its heads (a sum in another order may move a tie by one), and
    speculative output equals plain decoding on every rank."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = mp.get_context("spawn").Manager().dict()
    mp.spawn(_worker, args=(2, port, out), nprocs=2)
    for rank in range(2):
        got = out[rank]
        assert got["heads"] == 1 and got["codes"] <= 1 and got["scales"] < 1e-4
        assert got["spec_eq_plain"] and got["ranks_agree"]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_two_streams_at_once(fmt):
    """Calls in flight on two streams share no workspace: each gives what it gives alone."""
    from eagle4_b200 import ops
    from eagle4_b200.ops import native
    from eagle4_b200.ops.quant import kv_code, new_cache

    gen = torch.Generator(device="cuda").manual_seed(2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    calls = []
    for lens in ([3000, 17, 900, 5], [131, 4000, 2], [9000]):
        pages = -(-max(lens) // 16)
        kc, vc = (new_cache(len(lens) * pages * 16, 2, 128, torch.bfloat16, kv_code(fmt), "cuda") for _ in range(2))
        x = torch.randn(2, kc.shape[0], 2, 128, generator=gen, device="cuda")
        ops.kv_write(x[0], x[1], torch.arange(kc.shape[0], device="cuda"), kc, vc)
        table = torch.arange(len(lens) * pages, device="cuda").int().view(len(lens), pages)
        q = torch.randn(len(lens), 8, 128, generator=gen, device="cuda").to(torch.bfloat16)
        z = i32([0] * len(lens))
        calls.append((q, kc, vc, table, 16, i32(list(range(len(lens)))), z, i32(lens), z[:, None].contiguous(), z, 0.09,
                      max(lens)))
    want = [ops.attention(*c) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(ops.attention(*c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % len(calls)])
    native.check_errors()
