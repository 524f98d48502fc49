"""Head sizes that run as projections, then norm and RoPE: the projections' launch has nothing to
do with gammas and tables, whose rows are of another length than its 128-column blocks.  Tables
that fill their allocation to its last byte, and positions at their end."""
import numpy as np
import pytest
import torch

from conftest import Case, f32
from oracle import qkv_rope_oracle as orc

pytestmark = pytest.mark.gpu

ROWS = 131072  # x 80 or 96 values: whole multiples of 2 MiB, an allocation each


@pytest.mark.parametrize("D,hq,hkv", [(80, 32, 8), (96, 4, 4)])
@pytest.mark.parametrize("T", [61, 531, 1300])
def test_positions_at_the_end(device, D, hq, hkv, T):
    import mqk
    g = torch.Generator().manual_seed(T)
    pos = torch.randint(ROWS - 64, ROWS, (T,), generator=g, dtype=torch.int32)
    case = Case(T, 1, 512, hq, hkv, seed=T, head_dim=D, rows=ROWS, positions=pos)
    assert case.cos.numel() * 2 % 2 ** 21 == 0
    out = mqk.fused_qkv_rope(*case.args(device))
    torch.cuda.synchronize()
    idx = np.unique(np.linspace(0, T - 1, 9).astype(int))
    for name, o, r in zip("qkv", out, case.oracle(token_idx=idx, round_projection=True)):
        assert orc.rel_l2(f32(o).reshape(T, -1, D)[idx].reshape(r.shape), r) <= 1e-2, name
