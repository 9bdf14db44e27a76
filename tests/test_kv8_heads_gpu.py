"""The 8-bit attention with 5 to 8 query heads per kv head, and with thousands of rows in one call."""

import pytest
import torch

from eagle4_b200 import ops
from eagle4_b200.ops.quant import kv_code, new_cache

pytestmark = pytest.mark.gpu


def _cache(gen, slots, heads, dim, fmt):
    kc, vc = (new_cache(slots, heads, dim, torch.bfloat16, kv_code(fmt), "cuda") for _ in range(2))
    x = torch.randn(2, slots, heads, dim, generator=gen, device="cuda")
    ops.kv_write(x[0], x[1], torch.arange(slots, device="cuda"), kc, vc)
    return kc, vc


def _exact(q, kc, vc, req, ends, table, page, scale):
    """float64, rows that end at ``ends`` of their request's first positions; no extras."""
    t, hq, d = q.shape
    hk = kc.shape[1]
    n = int(ends.max())
    pos = torch.arange(n, device="cuda")
    out = torch.zeros(t, hq * d, dtype=torch.float64, device="cuda")
    for b in range(table.shape[0]):
        at = table[b].long()[pos // page] * page + pos % page
        k, v = (x.double() for x in ops.kv_read(kc, vc, at, torch.float32))
        for r in (req == b).nonzero().flatten().split(512):
            s = torch.einsum("rhgd,khd->rhgk", q[r].double().view(len(r), hk, -1, d), k) * scale
            s.masked_fill_(pos >= ends[r][:, None, None, None], -float("inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out[r] = torch.einsum("rhgk,khd->rhgd", p, v).reshape(len(r), -1)
    return out


def _near(got, want):
    # bf16's rounding (half of 2^-7 of the value's power of two) and 2^-12 of the weights each, of outputs up to the row's
    # largest; 2^-18: fp32 sums over up to 2^13 keys
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -12 + 2.0 ** -18) * want.abs().amax(-1, keepdim=True)
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float((got.double() - want).abs().max())}"


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hq,hk,d", [(64, 8, 128), (40, 8, 128), (12, 2, 64), (7, 1, 112)])
def test_five_to_eight_heads(fmt, hq, hk, d):
    """Every count of heads that two blocks share an SM for, in a batch that fills the GPU and rows alone: same bits."""
    from eagle4_b200.ops import native

    gen = torch.Generator(device="cuda").manual_seed(hq)
    lens = [(i * 2311) % 6000 for i in range(40)]
    page = 16
    pages = -(-max(lens) // page)
    kc, vc = _cache(gen, 40 * pages * page, hk, d, fmt)
    table = torch.randperm(40 * pages, generator=gen, device="cuda").int().view(40, pages)
    q = torch.randn(40, hq, d, generator=gen, device="cuda").to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ends, none = i32(lens), torch.zeros(40, dtype=torch.int32, device="cuda")
    req, ex = torch.arange(40, device="cuda").int(), torch.zeros(40, 1, dtype=torch.int32, device="cuda")
    got = ops.attention(q, kc, vc, table, page, req, none, ends, ex, none, d ** -0.5, 6000)
    _near(got, _exact(q, kc, vc, req, ends, table, page, d ** -0.5))
    for r in (1, 7, 23, 39):
        one = ops.attention(q[r:r + 1], kc, vc, table, page, req[r:r + 1], none[:1], ends[r:r + 1], ex[:1], none[:1],
                            d ** -0.5, 6000)
        assert torch.equal(one[0], got[r])
    native.check_errors()


@pytest.mark.parametrize("fmt,hq,hk,d,rows", [("fp8", 24, 4, 256, 2500), ("int8", 8, 1, 128, 4100), ("int8", 4, 2, 64, 3001)])
def test_a_prompt_of_thousands_of_rows(fmt, hq, hk, d, rows):
    """Two requests' prompts in one call, row i of each sees its first i + 1 positions (row 0's request: one of none)."""
    from eagle4_b200.ops import native

    gen = torch.Generator(device="cuda").manual_seed(rows)
    page = 16
    pages = -(-rows // page)
    kc, vc = _cache(gen, 2 * pages * page, hk, d, fmt)
    table = torch.randperm(2 * pages, generator=gen, device="cuda").int().view(2, pages)
    i = torch.arange(rows, device="cuda")
    req = (i >= rows // 3).int()
    ends = torch.where(req == 0, i, i - rows // 3 + 1).int()  # the first row sees nothing
    q = torch.randn(rows, hq, d, generator=gen, device="cuda").to(torch.bfloat16)
    none, ex = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    got = ops.attention(q, kc, vc, table, page, req, none, ends, ex, none, d ** -0.5, rows)
    assert not got[0].any()
    _near(got, _exact(q, kc, vc, req, ends, table, page, d ** -0.5))
    native.check_errors()


@pytest.mark.parametrize("hk,d,keys", [(1, 64, 50), (1, 256, 100), (8, 128, 3000)])
def test_between_projections(hk, d, keys):
    """GEMMs right before and after, which hold tensor memory too and start before their predecessor ends."""
    from eagle4_b200.ops import native

    gen = torch.Generator(device="cuda").manual_seed(d)
    kc, vc = _cache(gen, 4096, hk, d, "fp8")
    w = [torch.randn(n, k, generator=gen, device="cuda").mul_(0.05).to(torch.bfloat16)
         for n, k in ((4 * hk * d, 512), (512, 4 * hk * d))]
    x = torch.randn(1, 512, generator=gen, device="cuda").to(torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (torch.arange(256, device="cuda").int()[None], 16, i32(0), i32(0), i32(keys), i32(0)[None], i32(0), d ** -0.5, keys)

    def step():
        q = ops.linear(x, w[0]).view(1, 4 * hk, d)
        return ops.linear(ops.attention(q, kc, vc, *args), w[1])

    want = step().clone()
    torch.cuda.synchronize()
    for _ in range(100):
        got = step()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    native.check_errors()
