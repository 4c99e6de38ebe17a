"""Rows of experts at the ends of their ranges, in whole numbers, which every sum holds."""
import pytest
import torch

import fp6_llm_amd as fp6
from test_int4 import DEV, gpu

MANY = (1 << 24) + 3   # workgroups of 256 threads: more threads than a dimension of a grid has


def numbers(n, m):
    """[n, 8] of whole numbers that tell rows apart, in fp16."""
    t = torch.arange(n, device=DEV)
    return torch.stack([(t >> s) % m for s in range(0, 24, 3)], 1).half()


@gpu
def test_more_tokens_than_a_dimension_of_a_grid_has_workgroups():
    T, E = MANY, 3
    index = (torch.arange(T, dtype=torch.int32, device=DEV) * 7 % E).unsqueeze(1)
    x = numbers(T, 8)
    rows, plan = fp6.expert_sort(x, index, E)
    assert torch.equal(plan.order.long(), torch.sort(index[:, 0], stable=True).indices)
    assert torch.equal(rows, x[plan.order.long()])
    assert torch.equal(fp6.expert_combine(rows, plan, torch.full((T, 1), 3.0, device=DEV)), 3 * x)


@gpu
def test_gradients_of_more_tokens_than_a_dimension_of_a_grid_has_workgroups():
    T, k, E = MANY // 3 + 1, 9, 5   # (four experts of a token to a workgroup; torch itself indexes fewer than 2^26 rows)
    index = torch.arange(T * k, dtype=torch.int32, device=DEV).view(T, k) % E
    plan = fp6.expert_plan(index, E)
    rows = numbers(T * k, 4).requires_grad_()
    weights = (torch.arange(T * k, device=DEV) % 3).float().view(T, k).requires_grad_()
    grad = numbers(T, 8)
    got_rows, got_weights = torch.autograd.grad(fp6.expert_combine(rows, plan, weights), (rows, weights), grad)
    place = plan.place.long()
    assert torch.equal(got_rows[place].view(T, k, 8), weights.detach().half()[:, :, None] * grad[:, None])
    assert torch.equal(got_weights, (rows.detach()[place].view(T, k, 8) * grad[:, None]).float().sum(2))
