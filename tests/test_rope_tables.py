"""The rotary tables that device code keeps the addresses of."""

import torch

from eagle4_b200.ops import native


def test_angle_tables_stay_where_captured_graphs_read_them():
    dev = torch.device("cpu")
    first = native.rope_turns(64, 12345.0, dev)
    at, values = first.data_ptr(), first.clone()
    for i in range(200):
        native.rope_turns(64, 20000.0 + i, dev)
    again = native.rope_turns(64, 12345.0, dev)
    assert again is first and again.data_ptr() == at and torch.equal(again, values)
