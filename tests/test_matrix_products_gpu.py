"""Products of 11 bits on matrices whose roundings do not average: few entries, diagonals, few directions.  Against the formulas in 64
bits, within what their roundings can do (``half_bound``), and one rounding of the result."""
from __future__ import annotations

import math

import pytest
import torch

import _matrix_oracle as M
from fairscale_amd.optim import Muon, Precision, orthogonalize

pytestmark = pytest.mark.gpu

SHAPES = [(300, 300), (647, 1128), (1128, 647), (129, 2000)]
TYPES = [torch.float32, torch.bfloat16]


def generator(seed):
    return torch.Generator().manual_seed(seed)


def one_entry_a_row(shape, sizes, seed=0):
    """(matrix, (rows, columns)): sizes at random places of rows and columns of their own."""
    g = generator(seed)
    rows, cols = torch.randperm(shape[0], generator=g)[:len(sizes)], torch.randperm(shape[1], generator=g)[:len(sizes)]
    u = torch.zeros(shape)
    u[rows, cols] = torch.as_tensor(sizes, dtype=torch.float32)
    return u, (rows, cols)


ENTRIES = {"one": [0.37], "two": [1.0, 0.5825], "three": [1.0, -0.7, 0.1], "four": [0.3, -0.31, 0.9, 0.05], "five": [1.0, 1.0, -1.0, 1.0, 1.0], "all": None}


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("entries", ENTRIES)
def test_matrices_of_one_entry_in_a_row(entries, shape, dtype):
    sizes = ENTRIES[entries] or torch.ones(min(shape)).tolist()
    u, at = one_entry_a_row(shape, sizes)
    u = u.to(dtype)
    got = orthogonalize([u.cuda()], products="half")[0].cpu().double()
    x = u[at].double() / u.double().norm()
    want = M.orthogonal(u)[at]
    bound = torch.tensor([M.half_bound(v, v) for v in x.abs().unique().tolist()])[x.abs().unique(return_inverse=True)[1]]
    assert ((got[at] - want).abs() <= bound + want.abs() * (torch.finfo(dtype).eps / 2)).all()
    got[at] = 0.0
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["constant", "signs"])
def test_rank_one_with_entries_of_one_size(kind, shape, dtype):
    g = generator(1)
    side = lambda n: torch.randint(0, 2, (n,), generator=g) * 2.0 - 1.0 if kind == "signs" else torch.ones(n)
    u = (torch.outer(side(shape[0]), side(shape[1])) * 0.01).to(dtype)
    want = M.orthogonal(u)
    error = (orthogonalize([u.cuda()], products="half")[0].cpu().double() - want).norm().item()
    assert error <= M.half_bound(1.0, 1.0) + want.norm().item() * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_equal_rows(shape, dtype):
    """The gradient of a sum of outputs: rank one, entries of any size."""
    u = torch.randn(shape[1], generator=generator(2)).expand(shape).to(dtype)
    want = M.orthogonal(u)
    error = (orthogonalize([u.contiguous().cuda()], products="half")[0].cpu().double() - want).norm().item()
    assert error <= M.half_bound(1.0, 1.0, alike=False) + want.norm().item() * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 2, 5, 16])
def test_few_rows_that_are_not_zero(rows, dtype):
    """Rare tokens, idle experts.  Their singular values lie close to each other: every one is moved by no more than the bound."""
    u = torch.zeros(512, 1024)
    g = generator(rows)
    u[torch.randperm(512, generator=g)[:rows]] = torch.randn(rows, 1024, generator=g)
    u = u.to(dtype)
    x = torch.linalg.svdvals(u.double())[:rows] / u.double().norm()
    want = M.orthogonal(u)
    error = (orthogonalize([u.cuda()], products="half")[0].cpu().double() - want).norm().item()
    assert error <= math.sqrt(rows) * M.half_bound(x.min().item(), x.max().item(), alike=False) + want.norm().item() * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("coefficients, steps", [(M.COEFFICIENTS, 6), (M.COEFFICIENTS, 10), ((4.0848, -6.8946, 2.9270), 5), ((4.0848, -6.8946, 2.9270), 3)], ids=str)
def test_iterations_that_multiply_the_error_take_22_bits(coefficients, steps):
    us = [torch.randn(300, 500, generator=generator(4)).cuda(), one_entry_a_row((300, 500), ENTRIES["four"])[0].cuda()]
    half, split = (orthogonalize(us, products=p, steps=steps, coefficients=coefficients) for p in ("half", "split"))
    assert all(torch.equal(a, b) for a, b in zip(half, split))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_steps_of_parameters_without_masters(dtype):
    """The default there is 11 bits.  From zero, without momentum and decay, the parameter is the orthogonalised gradient."""
    shape, sizes = (300, 400), ENTRIES["three"]
    u, at = one_entry_a_row(shape, sizes)
    p = torch.nn.Parameter(torch.zeros(shape, dtype=dtype, device="cuda"))
    opt = Muon([p], lr=1.0, weight_decay=0.0, momentum=0.0, precision=Precision.MEMORY_EFFICIENT_MIXED_PRECISION)
    p.grad = u.to(dtype).cuda()
    opt.step()
    got, want = p.detach().cpu().double(), -M.orthogonal(u.to(dtype))
    for k, (i, j) in enumerate(zip(*at)):
        x = abs(u.to(dtype)[i, j].double() / u.to(dtype).double().norm()).item()
        assert abs(got[i, j] - want[i, j]) <= M.half_bound(x, x) + abs(want[i, j]) * (torch.finfo(dtype).eps / 2 + 3 * 2**-24)
    got[at] = 0.0
    assert (got == 0).all()
