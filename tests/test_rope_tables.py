"""Rotary tables that device code keeps the addresses of, and the shapes that positions come in."""

from types import SimpleNamespace

import pytest
import torch

from eagle4_b200 import ops
from eagle4_b200.ops import native
from eagle4_b200.ops.quant import kv_code, new_cache


def test_angle_tables_stay_where_captured_graphs_read_them():
    dev = torch.device("cpu")
    first = native.rope_turns(64, 12345.0, dev)
    at, values = first.data_ptr(), first.clone()
    for i in range(200):
        native.rope_turns(64, 20000.0 + i, dev)
    again = native.rope_turns(64, 12345.0, dev)
    assert again is first and again.data_ptr() == at and torch.equal(again, values)


def _cfg(sections):
    return SimpleNamespace(num_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=32, rope_theta=1e6, rms_norm_eps=1e-6,
                           rope_sections=sections, rope_interleaved=False, attn_output_gate=False, norm_offset=False)


def _prepare(pos, sections, kv, device, dtype=torch.bfloat16):
    t = pos.shape[-1]
    qkv = torch.randn(t, 8 * 64, generator=torch.Generator().manual_seed(t)).to(dtype).to(device)
    kc, vc = (new_cache(t, 2, 64, dtype, kv_code(kv), device) for _ in range(2))
    q, _ = ops.qkv_prepare(qkv, _cfg(sections), pos.to(device), torch.arange(t, device=device), kc, vc, None, None)
    rows = kc if kv == "bf16" else ops.kv_read(kc, vc, torch.arange(t, device=device), torch.float32)[0]
    return q, rows


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("sections", [None, (4, 6, 6)])
def test_one_axis_as_a_row(device, kv, sections):
    """Positions [1, T] turn like positions [T], whatever the config's sections are."""
    pos = torch.tensor([0, 7, 1000, 3, 90000])
    for a, b in zip(_prepare(pos, sections, kv, device), _prepare(pos[None], sections, kv, device)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_one_row_of_a_transposed_table(device, kv):
    """A decode step's positions [axes, 1] cut from a table [rows, axes]: the strides of one element mean nothing."""
    table = torch.tensor([[5, 900, 31], [6, 17, 2]], device=device)
    for a, b in zip(_prepare(table[:1].t(), (4, 6, 6), kv, device),
                    _prepare(torch.tensor([[5], [900], [31]]), (4, 6, 6), kv, device)):
        assert torch.equal(a, b)
