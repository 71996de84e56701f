"""The feed-forward operators at the ends of their ranges: hidden layers whose rows are 2^27 bytes apart, values far from one, more rows than one launch has threads."""
import math

import pytest
import torch

import feed_forward_oracle as oracle
from kutacc_amd import capi
from test_gpu_feed_forward import BF16, FP32, Room, cpu_randn, ok

pytestmark = pytest.mark.gpu


def test_gated_transition_of_a_hidden_layer_whose_rows_are_far_apart():
    """32 rows of 69.4 million hidden units, the last of them 2^32 bytes behind the first: down_w picks units at both ends and around a power of two, so that every row's
    result is a sum of few, its own."""
    rows, c_o, c_i = 32, 8, (1 << 32) // (2 * 31) // 8 * 8 + 4096
    picked = [0, 1, (1 << 23) - 1, 1 << 23, c_i // 2, c_i - 8, c_i - 1, c_i - 4096]
    x = cpu_randn(1, rows, c_o)
    w = [cpu_randn(2, len(picked), c_o), cpu_randn(3, len(picked), c_o), cpu_randn(4, c_o, len(picked))]
    gpu = [torch.ones(c_i, c_o, device="cuda", dtype=BF16) for _ in range(2)] + [torch.zeros(c_o, c_i, device="cuda", dtype=BF16)]
    gpu[0][picked], gpu[1][picked], gpu[2][:, picked] = w[0].cuda(), w[1].cuda(), w[2].cuda()
    out = Room(rows, c_o, BF16)
    ok(capi.GatedTransition(x.cuda(), *gpu, out.view))
    want, off = oracle.gated_transition(x, *w, "silu")["out"]
    # (the bound is of the units that are picked: the others are zeros times their values, and add nothing)
    oracle.close(out.view, want, oracle.stored(want, off, BF16), "out")
    out.untouched("out")
