"""``torchmatch_amd.attention.ops`` has every op of its namespace, under its name."""

from __future__ import annotations

import torch

from torchmatch_amd.attention import ops


def test_every_registered_op_is_there():
    names = {n.split("::")[1].split(".")[0] for n in torch._C._dispatch_get_all_op_names()
             if n.startswith("attention::")}
    assert len(names) >= 8 and names == set(ops.__all__)
    for name in names:
        assert getattr(ops, name) is getattr(torch.ops.attention, name)
