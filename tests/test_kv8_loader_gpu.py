"""The 8-bit attention's loading warps: a chunk's keys may be context and extras in one warp, mapped and unmapped."""

import pytest
import torch

from eagle4_b200 import ops
from eagle4_b200.ops.quant import kv_code, new_cache

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hq,hk,d", [(6, 1, 256), (4, 2, 64)])
def test_every_lane_reads_its_own_keys_cell(fmt, hq, hk, d):
    """The same keys with the last 0 to 128 of them as extras instead of context, in rows of two requests whose chunks
    follow each other in one block: each lane's cell of a chunk, and of the chunk before, holds another address, so a
    lane that read a neighbour's old cell would take another key."""
    from eagle4_b200.ops import native

    gen = torch.Generator(device="cuda").manual_seed(3)
    page, pages = 7, 80
    kc, vc = (new_cache(2 * pages * page, hk, d, torch.bfloat16, kv_code(fmt), "cuda") for _ in range(2))
    x = torch.randn(2, 2 * pages * page, hk, d, generator=gen, device="cuda")
    ops.kv_write(x[0], x[1], torch.arange(2 * pages * page, device="cuda"), kc, vc)
    bt = torch.randperm(2 * pages, generator=gen, device="cuda").int().view(2, pages)
    slot = lambda b, n: bt[b].long()[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page  # noqa: E731
    lens = [(r * 37) % 400 + 129 for r in range(129)]
    q = torch.randn(2, hq, d, generator=gen, device="cuda").to(torch.bfloat16)[torch.arange(129) % 2].contiguous()
    req = _i32([r % 2 for r in range(129)])
    ex = torch.zeros(129, 128, dtype=torch.int32, device="cuda")
    for r, n in enumerate(lens):
        ex[r, :r] = slot(r % 2, n)[n - r:].int()
    args = (bt, page, req, _i32([0] * 129))
    split = lambda: ops.attention(q, kc, vc, *args, _i32([n - r for r, n in enumerate(lens)]), ex,  # noqa: E731
                                  _i32(list(range(129))), d ** -0.5, 640)
    want = ops.attention(q, kc, vc, *args, _i32(lens), ex, _i32([0] * 129), d ** -0.5, 640)
    for _ in range(20):
        assert torch.equal(split(), want)
    native.check_errors()


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_lengths_past_the_bound_are_reported(fmt):
    """A row longer than ``max_keys`` says, up to the largest length an int32 holds: the error word, the other rows as
    they are, and nothing read past the row's block table."""
    from eagle4_b200.ops import native

    kc, vc = (new_cache(64, 2, 64, torch.bfloat16, kv_code(fmt), "cuda") for _ in range(2))
    x = torch.randn(64, 2, 64, device="cuda")
    ops.kv_write(x, x, torch.arange(64, device="cuda"), kc, vc)
    q = torch.randn(3, 4, 64, device="cuda").to(torch.bfloat16)
    call = lambda start, end, keys: ops.attention(q, kc, vc, _i32([[0, 1, 2, 3]]), 16, _i32([0] * 3), _i32(start), _i32(end),  # noqa: E731
                                                  _i32([[0]] * 3), _i32([0] * 3), 0.1, keys)
    want = call([0, 0, 0], [50, 0, 17], 64)
    native.check_errors()
    top = 2 ** 31 - 1
    for start, end in ((0, top), (-top, top), (-top - 1, 5), (0, 300)):
        got = call([0, start, 0], [50, end, 17], 64)
        with pytest.raises(RuntimeError, match="error code"):
            native.check_errors()
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    with pytest.raises(RuntimeError, match="too many keys"):
        call([0] * 3, [1] * 3, 2 ** 31)
    native.check_errors()
