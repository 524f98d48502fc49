"""How much memory and how many workgroups the paged operators ask for (no GPU needed)."""
from __future__ import annotations

import pytest
import torch

from test_paged_ops_host import WORKSPACE, attn, cache, lib, ref, select  # noqa: F401

# (a call that is not refused would launch on these addresses)
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that no GPU may be given")
MB = 1 << 20


@pytest.mark.parametrize("D,Hkv", [(128, 8), (64, 40), (256, 4)])
def test_room_of_short_sequences(lib, D, Hkv):  # noqa: F811
    """Partial results: two a workgroup of 256, 32 rows each, whatever the number of sequences."""
    size = lambda n, T: lib.mqk_paged_attn_workspace_size(ref(cache(n_seqs=n, bt_cols=4096, Hkv=Hkv, D=D)), T, 4 * Hkv, 0, 0)
    most = 2 * 256 * (32 * (D + 2) * 4 + 64) + MB
    assert 0 < size(3, 3) <= size(16384, 16384) <= size(16384, 8 * 16384) <= most


def test_room_of_packed_sequences(lib):  # noqa: F811
    """The same beside the long sequences' (two a place of 512, 128 rows each)."""
    size = lambda n, T: lib.mqk_paged_attn_workspace_size(ref(cache(n_seqs=n, bt_cols=4096, Hkv=8)), T, 32, 1, 0)
    most = 2 * 256 * (32 * 130 * 4 + 64) + 2 * 512 * (128 * 130 * 4 + 64) + MB
    assert 0 < size(3, 3) <= size(64, 2048) <= size(16384, 16384) <= most


@pytest.mark.parametrize("T,cols,Hkv", [(2048, 2560, 8), (8192, 8192, 8), (64, 65536, 8), (1 << 18, 4096, 8), (1000, 30001, 1)])
def test_room_of_a_selection(lib, T, cols, Hkv):  # noqa: F811
    """Tokens are taken in rounds: 256 MiB of scores at most."""
    size = lib.mqk_paged_select_workspace_size(ref(cache(bt_cols=cols, Hkv=Hkv)), T)
    assert 0 < size <= 256 * MB + 128 * 1024


def test_selection_of_long_prompts(lib):  # noqa: F811
    """64 prompts of 4096 tokens in tables of 4096 pages: many rounds, not too much work."""
    c = dict(n_seqs=64, bt_cols=4096, Hkv=8, num_blocks=1 << 20, k=None, v=None)
    assert select(lib, T=64 * 4096, cache=cache(**c)) == WORKSPACE


def test_packed_steps_of_many_sequences(lib):  # noqa: F811
    """Sequences without a chunk have no workgroups in the chunks' launch: a step of 2^20 is not too
    much work for one."""
    assert attn(lib, T=1 << 20, Hq=16, cu=1 << 20, cache=cache(n_seqs=1 << 20, Hkv=16, bt_cols=100)) == WORKSPACE
