"""The products of the matrix operators: 11 bits on matrices whose roundings do not average (few entries, diagonals, few directions),
against the formulas in 64 bits within what the roundings can do (``half_bound``); other steps and coefficients; lists that
go through the workspace in parts."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import _matrix_oracle as M
from fairscale_amd import _cabi
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


# ---- steps and coefficients through the launches of larger matrices ------------------------------------------------------

ITERATIONS = [(M.COEFFICIENTS, 1), (M.COEFFICIENTS, 2), (M.COEFFICIENTS, 3), (M.COEFFICIENTS, 4), (M.COEFFICIENTS, 10), ((1.5, -0.5, 0.0), 8), ((1.875, -1.25, 0.375), 6),
              ((0.0, 0.0, 0.0), 2), ((-3.4445, 4.7750, -2.0315), 3), ((2.0, -1.5, 0.5), 12), ((8.0, 0.0, 0.0), 3), ((1.0, 0.0, 0.0), 4)]


def allowed(products, steps, longest):
    """Simulated with these roundings (steps in pairs with 22 bits), every iteration above is off by at most 1.3e-6 with 22 bits and 4e-3
    (ten of the usual steps) or 1.3e-3 (the others) with 11; twice 2.6e-6 and 1.9e-3 are allowed for up to five steps, in proportion for
    more.  Sums of l terms add 3 l / 32 roundings of 2^-24 in Gram matrices, and the result is rounded once."""
    return 2**-24 + max(1, steps / 5) * ({"split": 2 * 2.6e-6, "half": 2 * 1.9e-3}[products] + 3 * longest / 32 * 2**-24)


@pytest.mark.parametrize("products", ["split", "half"])
@pytest.mark.parametrize("coefficients, steps", ITERATIONS, ids=str)
def test_other_steps_and_coefficients_of_matrices_of_many_tiles(coefficients, steps, products):
    """Even and odd numbers of steps, so that a pair and a single step come last; wide, tall, with a split Gram matrix, in LDS."""
    us = [torch.randn(*s, generator=generator(sum(s))) for s in ((300, 500), (500, 300), (130, 4100), (2, 140, 200), (90, 140))]
    for u, o in zip(us, orthogonalize([u.cuda() for u in us], products=products, steps=steps, coefficients=coefficients)):
        for x, y in zip(o.reshape(-1, *o.shape[-2:]), M.orthogonal(u, steps, coefficients).reshape(-1, *o.shape[-2:])):
            assert M.relative(x, y) <= allowed(products, steps, max(u.shape[-2:])), tuple(u.shape)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("products", ["split", "half"])
def test_muon_steps_of_other_numbers_of_products(steps, products):
    params = [torch.nn.Parameter(torch.randn(*s, generator=generator(1)).cuda()) for s in ((300, 500), (500, 300), (40, 60))]
    before = [p.detach().double().cpu() for p in params]
    opt = Muon(params, lr=0.05, ns_steps=steps, products=products)
    for k, p in enumerate(params):
        p.grad = torch.randn(p.shape, generator=generator(k + 5)).cuda()
    opt.step()
    for p, w in zip(params, before):
        want, _ = M.step(w, p.grad, torch.zeros(p.shape), lr=0.05, steps=steps)
        moved = (want - w * (1 - 0.05 * 0.1)).norm().item()
        # the parameter's own arithmetic: three roundings of fp32
        assert (p.detach().double().cpu() - want).norm().item() <= 3 * 2**-24 * want.norm().item() + moved * allowed(products, steps, max(p.shape))


# ---- lists that go through the workspace in parts ---------------------------------------------------------------------------

@pytest.mark.parametrize("products, batch", [("split", 12), ("half", 20)])
def test_a_batch_that_is_cut_by_the_workspace(products, batch):
    """Five matrices and a batch whose intermediates pass 4 GiB together: the cut falls inside the batch.  All have contents of their own,
    the batch's are slices of columns in larger rows, on both sides, and each gives the bits it gives alone."""
    n, wide = 4096, 4104
    base = torch.randn(batch, n, wide, device="cuda", generator=torch.Generator("cuda").manual_seed(3), dtype=torch.bfloat16)
    us = [torch.randn(n, n, device="cuda", generator=torch.Generator("cuda").manual_seed(10 + k), dtype=torch.bfloat16) for k in range(5)]
    us.append(base[:, :, 5:5 + n])
    into = torch.full((batch, n, wide), 7.0, device="cuda", dtype=torch.bfloat16)
    outs = [torch.empty_like(u) for u in us[:5]] + [into[:, :, 2:2 + n]]

    def needed(list_of):
        rows = (_cabi.FsMatrix * len(list_of))()
        for row, u in zip(rows, list_of):
            row.src = row.dst = 1 << 20
            row.batch, row.rows, row.cols = u.numel() // (n * n), n, n
            row.src_ld = row.dst_ld = n
            row.src_stride = row.dst_stride = n * n
        size = ctypes.c_int64()
        options = _cabi.FsOrthOptions(*M.COEFFICIENTS, 1e-7, 5, {"half": _cabi.PRODUCTS_HALF, "split": _cabi.PRODUCTS_SPLIT}[products])
        _cabi.check(_cabi.lib().fsadam_orth_workspace(rows, len(list_of), ctypes.byref(options), ctypes.byref(size)))
        return size.value

    one = needed(us[:1])
    assert (5 + batch) * one > 4 << 30 >= needed(us) and 6 * one < 4 << 30, "two parts, the second begins inside the batch"
    got = orthogonalize(us, products=products, out=outs)
    for u, o in zip(us[:5], got):
        assert torch.equal(o, orthogonalize([u], products=products)[0])
    for k in range(batch):
        assert torch.equal(got[5][k], orthogonalize([base[k, :, 5:5 + n].contiguous()], products=products)[0]), k
    assert (into[:, :, :2] == 7.0).all() and (into[:, :, 2 + n:] == 7.0).all()


def test_a_step_whose_batch_is_cut_by_the_workspace():
    """Masters, gradients, momenta and copies of one parameter of 14 matrices: each bit as from 14 parameters of their own."""
    n, batch = 4096, 14
    g = torch.Generator("cuda").manual_seed(5)
    whole = torch.nn.Parameter(torch.randn(batch, n, n, device="cuda", generator=g, dtype=torch.float16) * 0.02)
    opt = Muon([whole], lr=0.05, adjust_lr_fn="match_rms_adamw")
    assert opt.products == "split"
    whole.grad = torch.randn(batch, n, n, device="cuda", generator=g, dtype=torch.float16)
    opt.state[whole]["momentum_buffer"] = torch.randn(batch, n, n, device="cuda", generator=g) * 0.5
    before = [whole.detach().clone(), opt.state[whole]["momentum_buffer"].clone()]
    opt.step(scale=2.0)
    for k in range(batch):
        p = torch.nn.Parameter(before[0][k].clone())
        one = Muon([p], lr=0.05, adjust_lr_fn="match_rms_adamw")
        one.state[p]["momentum_buffer"] = before[1][k].clone()
        p.grad = whole.grad[k].clone()
        one.step(scale=2.0)
        assert torch.equal(whole[k], p) and torch.equal(opt.state[whole]["master"][k], one.state[p]["master"]), k
        assert torch.equal(opt.state[whole]["momentum_buffer"][k], one.state[p]["momentum_buffer"]), k
