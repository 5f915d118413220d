"""The sizes in operator_cases reach the kernels that they are there for, and
every kernel that the operators' rules can choose."""
import random

import pytest
import torch

import operator_cases as cases
from dfsattn_amd import _lib, ops

BF = torch.bfloat16


@pytest.mark.parametrize("m,n,k,form", cases.LINEAR)
def test_linear_cases_take_their_form(m, n, k, form):
    assert cases.linear_form(m, n, k) == form


@pytest.mark.parametrize("B,H,G,L,S,D,left,right,sinks,rolling,form", cases.WINDOW)
def test_window_cases_take_their_form(B, H, G, L, S, D, left, right, sinks, rolling, form):
    assert cases.window_form(B, H, G, L, S, D, left, right, sinks, rolling, BF) == form


def test_every_form_that_sizes_can_choose_has_a_case():
    rng = random.Random(0)
    listed = {c[-1] for c in cases.LINEAR}
    for _ in range(60000):
        m, n, k = (int(2 ** rng.uniform(0, e)) for e in (13, 15, 14))
        if rng.random() < 0.6:
            n, k = max(8, n // 8 * 8), max(8, k // 8 * 8)
        assert cases.linear_form(m, n, k, k % 8 == 0 and rng.random() < 0.8) in listed, (m, n, k)
    listed = {c[-1] for c in cases.WINDOW}
    for _ in range(20000):
        G = rng.choice([1, 2, 3, 8, 20])
        H, L, S = G * rng.choice([1, 2, 4]), int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 14))
        left, right = (rng.choice([None, int(2 ** rng.uniform(0, 12))]) for _ in range(2))
        form = cases.window_form(rng.choice([1, 3, 16, 64]), H, G, L, S, rng.choice([64, 128]), left, right,
                                 rng.choice([0, 70]), False, BF)
        assert form in listed, (G, H, L, S, left, right)


def test_forms_refuse_sizes_that_are_not_positive():
    for sizes in ((0, 1, 1), (1, -1, 1), (1, 1, 0)):
        assert _lib.lib().dfs_linear_form(*sizes, 1) == -1
    assert _lib.lib().dfs_window_attention_form(bytes(_lib.WindowArgs())) == -1
    assert _lib.lib().dfs_window_attention_form(None) == -1
