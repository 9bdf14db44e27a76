"""How many bits the 8-bit digits of queries and softmax weights carry, where no averaging hides a lost digit.

Attention over an 8-bit cache cuts a query (per head, its largest element's power of two at full scale) and each chunk's
weights (the largest at full scale) into three digits: e4m3, each of the remainder times 16 (2^-12 relative), or int8,
base 256 of a 23-bit fixed-point number. Two keys whose rows are constant over the head dim make every element's and
every weight's error fall into the output undiminished."""

import pytest
import torch

from eagle4_b200 import ops
from eagle4_b200.ops.quant import kv_code, new_cache

D, HEADS, ROWS = 64, 8, 64
VALUE = 1.96875  # outputs near two, where fp16's half unit is 2^-12 of them


def _cut(x, fmt, terms):
    """``x`` in units of its full scale (1 / 2 at most for queries, 1 for weights), from its first ``terms`` digits."""
    if fmt == "fp8":
        y, out = x * 2.0 ** 8, torch.zeros_like(x)
        for t in range(terms):
            d = y.float().to(torch.float8_e4m3fn).double()
            out += d * 16.0 ** -t
            y = (y - d) * 16
        return out * 2.0 ** -8
    n = (x * 2.0 ** 22).round()
    drop = 256.0 ** (3 - terms)
    return (n / drop).round() * drop * 2.0 ** -22


def _case(opposite):
    """Queries (constant over the head dim) with 11 random bits, scores +S and -S for S in 0.4 .. 0.8, values of one sign
    or two."""
    gen = torch.Generator().manual_seed(5)
    q = ((torch.randint(1024, 2048, (ROWS, HEADS), generator=gen) / 1024.0)[..., None].expand(-1, -1, D)).half()
    k = torch.ones(2, 1, D) * torch.tensor([1.0, -1.0]).view(2, 1, 1)
    v = torch.full((2, 1, D), VALUE) * torch.tensor([1.0, -1.0 if opposite else 1.0]).view(2, 1, 1)
    return q.contiguous(), k, v, 0.4 / D


def _cached(k, v, fmt, device="cpu"):
    kc, vc = (new_cache(16, 1, D, torch.float16, kv_code(fmt), device) for _ in range(2))
    at = torch.arange(2, device=device)
    ops.kv_write(k.to(device), v.to(device), at, kc, vc)
    return kc, vc, [x.cpu().double()[:, 0] for x in ops.kv_read(kc, vc, at, torch.float32)]


def _out(q, kv, scale, fmt, q_terms=None, w_terms=None):
    k, v = kv
    x = q.double()
    if q_terms is not None:
        full = 2.0 ** (torch.floor(torch.log2(x.abs().amax(-1, keepdim=True))) + 1)
        x = _cut(x / full, fmt, q_terms) * full
    p = torch.exp2(torch.einsum("rhd,kd->rhk", x, k) * scale / torch.log(torch.tensor(2.0, dtype=torch.float64)))
    b = v.abs().amax(-1)  # what the value scales weigh the maximum by (equal here)
    w = p * b / (p * b).amax(-1, keepdim=True)
    cut = w if w_terms is None else _cut(w, fmt, w_terms)
    return torch.einsum("rhk,kd->rhd", cut, v / b[:, None]) / (w / b).sum(-1, keepdim=True)


def _bad(got, want):
    # fp16's half unit; 2^-12 of a query's element (score up to 0.8, the output moves by at most 0.45 of it) and of a
    # weight (at most one half of the sum); fp32 arithmetic
    half_unit = torch.exp2(torch.floor(torch.log2(want.abs())) - 11)
    tol = half_unit + (0.45 + 0.5) * 2.0 ** -12 * VALUE + 2.0 ** -18
    return ((got.double() - want).abs() > tol).sum().item()


@pytest.mark.parametrize("opposite", [False, True])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_the_bound_notices_a_lost_digit(fmt, opposite):
    """The bound the kernel is held to below, on the model: three digits pass, fewer do not (an int8 digit is 8 bits, so
    fp16 outputs cannot tell two from three)."""
    q, k, v, scale = _case(opposite)
    kv = _cached(k, v, fmt)[2]
    want = _out(q, kv, scale, fmt)
    few = 2 if fmt == "fp8" else 1
    assert _bad(_out(q, kv, scale, fmt, 3, 3).half(), want) == 0
    assert _bad(_out(q, kv, scale, fmt, 3, few).half(), want) > 0
    if opposite:
        assert _bad(_out(q, kv, scale, fmt, few, 3).half(), want) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("opposite", [False, True])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_queries_and_weights_carry_three_digits(fmt, opposite):
    from eagle4_b200.ops import native

    q, k, v, scale = _case(opposite)
    kc, vc, kv = _cached(k, v, fmt, "cuda")
    i32 = lambda x: torch.full((ROWS,), x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.attention(q.cuda(), kc, vc, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 16, i32(0), i32(0), i32(2),
                        i32(0)[:, None], i32(0), scale, 2).view(ROWS, HEADS, D)
    native.check_errors()
    assert _bad(got.cpu(), _out(q, kv, scale, fmt)) == 0
