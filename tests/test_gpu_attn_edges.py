"""Attention over the paged 4-bit cache where sizes of values, windows and divided contexts go to their ends, against the 64-bit
definitions of kv_data.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_data as kd
from flintnsteel_amd import ops
from test_gpu_attn_half import MANY_ROWS, Setup, _check_attn, _rand

pytestmark = pytest.mark.gpu


def _upload(s: Setup) -> None:
    s.cache.pages.copy_(torch.from_numpy(s.host.raw.copy()).view(s.cache.pages.shape))
    s.batch.page_table.copy_(torch.from_numpy(s.table))


# ---- windows ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30, 3])
def test_windows_of_any_width_where_a_sequence_has_fewer_positions_than_new_tokens(window, many, dtype):
    """Tokens before position 0 see nothing, the others what the window leaves them."""
    s = Setup([20, 70], [20, 70], 16, 1, 64, seed=83, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else 70
    s.kv_lens = [5, 67]
    s.batch.kv_len.copy_(torch.tensor(s.kv_lens, dtype=torch.int32))
    _, out = _check_attn(s, 1, dtype, window=window)
    assert (out[:15] == 0).all() and (out[15:20] != 0).any(-1).all()
    assert (out[20:23] == 0).all() and (out[23:90] != 0).any(-1).all()
