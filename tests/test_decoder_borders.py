"""Which tokens a row of logits keeps (``mlc.ops.sample``): rows whose borders lie where a kernel
can miss them, against the definition in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import decoder_reference as ref
from mlc import ops
from test_decoder_operators import NEAR, TYPES, normal, options_of

gpu = pytest.mark.gpu
INF = float("inf")


# --------------------------------------------------------------------------
# the tokens that a row keeps
# --------------------------------------------------------------------------

def check_shares(row, n, **given):
    """``n`` random numbers, evenly over [0, 1), for one row: that the tokens are the right ones
    says which are kept and with which shares, as one draw does not."""
    uniform = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float()
    got = ops.sample(row.expand(n, -1), uniform.cuda(), **options_of(n, **given)).cpu().numpy()
    at, w = ref.kept(row.double().cpu().numpy(), **given)
    sums, u = np.cumsum(w), uniform.double().numpy()
    place = np.searchsorted(sums, u * sums[-1], side="right").clip(max=len(at) - 1)
    edges = np.concatenate([[-1.0], sums[:-1] / sums[-1], [2.0]])
    margin = np.minimum(u - edges[place], edges[place + 1] - u)
    wrong = (got != at[place]) & (margin > NEAR)
    assert not wrong.any(), (int(wrong.sum()), n, got[wrong][:5], at[place][wrong][:5], margin[wrong][:5])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", (1025, 1031, 2044, 4099, 8193, 8199, 50256, 50257, 50260, 50263, 50265))
def test_rows_whose_likely_tokens_lie_behind_the_last_whole_pack(dtype, size):
    """A token of the row's end, where it is no multiple of eight, at a border or in front of it: an
    end of text that is likely."""
    for rank in (1, 2, 5, 20, 50):
        x = normal(size, dtype=dtype, seed=rank, spread=3.0)
        other = x.float().argsort(descending=True, stable=True)[rank - 1].item()
        last = size - 1 - rank % max(1, size % 8)
        x[[last, other]] = x[[other, last]]
        for top_k in (2, 50, 512):
            for given in ({}, {"top_p": 0.9}, {"min_p": 0.01}, {"temperature": 0.8, "top_p": 0.95, "min_p": 0.002}):
                check_shares(x, 257, top_k=top_k, **given)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_tokens_take_nothing_of_their_neighbours(dtype):
    """A weight of 2^-41, half a step, beside masked tokens, at the random number 0."""
    x = torch.full((1, 3000), -INF, dtype=dtype, device="cuda")
    x[0, 8], x[0, 2992] = -41.0, 0.0
    for given in ({}, {"top_k": 2000}, {"top_k": 600, "min_p": 0.0}):
        # the temperature is log2 e, so that the weight is 2^-41
        options = options_of(1, temperature=1.4426950408889634, **given)
        assert ops.sample(x, torch.zeros(1, device="cuda"), **options).item() in (8, 2992)
