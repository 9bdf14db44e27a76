"""The accepted rows' moves in 16-bit KV caches (the 8-bit ones are in test_kv8_gpu.py)."""

import pytest
import torch

from eagle4_b200 import ops


def _moves(gen, requests, rows, span):
    """Per request an ascending path of ``rows`` of ``span`` rows moves to the first positions: [0, 2, 5, ...]."""
    src, dst = [], []
    for b in range(requests):
        path = torch.randperm(span, generator=gen)[:rows].sort().values.tolist()
        src += [b * span + r for r in path]
        dst += [b * span + i for i in range(rows)]
    return src, dst


def _expect(c, src, dst):
    want = c.clone()
    for s, d in zip(src, dst):
        if s >= 0 and d >= 0:
            want[d] = c[s]
    return want


def test_negative_slots_move_nothing_on_cpu():
    kc, vc = (torch.arange(6 * 8).float().view(6, 1, 8) + i for i in range(2))
    src, dst = [-1, 2, 4, -3], [3, -1, 1, -2]
    want = [_expect(c, src, dst) for c in (kc, vc)]
    ops.kv_commit([kc], [vc], torch.tensor(src), torch.tensor(dst))
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("layers,heads,dim,requests,rows,span", [
    (16, 4, 256, 1, 6, 16), (3, 8, 128, 8, 20, 64), (70, 1, 64, 40, 16, 50), (2, 3, 24, 1, 1000, 3000)])
def test_moves_read_their_sources_before_other_moves_overwrite_them(layers, heads, dim, requests, rows, span):
    """Every move's source as it was before the call, though other moves of the call write onto it: the blocks that
    copy rows run in no order."""
    from eagle4_b200.ops import native

    gen = torch.Generator().manual_seed(layers * dim)
    src, dst = _moves(gen, requests, rows, span)
    src += [-1, 7]
    dst += [5, -1]
    caches = [torch.randn(requests * span, heads, dim, generator=gen).to(torch.bfloat16).cuda() for _ in range(2 * layers)]
    want = [_expect(c, src, dst) for c in caches]
    s, d = (torch.tensor(x, device="cuda") for x in (src, dst))
    ops.kv_commit(caches[:layers], caches[layers:], s, d)
    native.check_errors()
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


@pytest.mark.gpu
def test_moves_go_to_the_caches_of_the_call():
    """Calls that share the K cache and differ in the V cache, or in a cache that took a freed one's address."""
    k, v1, v2 = (torch.randn(8, 2, 64, device="cuda").to(torch.bfloat16) for _ in range(3))
    s, d = torch.tensor([5], device="cuda"), torch.tensor([1], device="cuda")
    kept = v1.clone()
    kept[1] = v1[5]
    ops.kv_commit([k], [v1], s, d)
    want = _expect(v2, [5], [1])
    v1[5] = 0
    ops.kv_commit([k], [v2], s, d)
    assert torch.equal(v2, want) and torch.equal(v1[:5], kept[:5])


@pytest.mark.gpu
def test_refusals_and_bounds():
    from eagle4_b200.ops import native

    c = torch.zeros(8, 2, 64, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([1], device="cuda")
    with pytest.raises(RuntimeError, match="one type and shape"):
        ops.kv_commit([c], [torch.zeros(8, 2, 32, device="cuda", dtype=torch.bfloat16)], at, at + 1)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.kv_commit([c], [torch.zeros(8, 4, 64, device="cuda", dtype=torch.bfloat16)[:, :2]], at, at + 1)
    with pytest.raises(RuntimeError, match="multiple of 16 bytes"):
        ops.kv_commit([torch.zeros(8, 1, 4, device="cuda", dtype=torch.bfloat16)] * 2,
                      [torch.zeros(8, 1, 4, device="cuda", dtype=torch.bfloat16)] * 2, at, at + 1)
    ops.kv_commit([], [], at, at)
    ops.kv_commit([c], [c.clone()], at[:0], at[:0])
    native.check_errors()
    ops.kv_commit([c], [c.clone()], at, at + 100)  # past the cache: reported, not written
    with pytest.raises(RuntimeError, match="error code"):
        native.check_errors()
