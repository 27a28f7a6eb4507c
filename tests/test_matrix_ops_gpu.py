"""The matrix operators on the GPU against the same formulas in 64 bits.

Tolerances.  A rounding to a type is off by at most ``finfo.eps / 2`` of the value.  ``orthogonalize`` adds the error of its products:
with ``"half"`` the operands carry 11 bits, and a simulation of the iteration with these roundings against 64 bits
gives at most 1.9e-3 of the result's norm over Gaussian matrices, matrices of low rank with noise and decaying
spectra (sizes 64 to 2304); with ``"split"`` at most 2.6e-6 for Gaussian ones and 3e-5 for the others, where
fp32 products give the same.  Twice these are allowed, plus the rounding of the result.  (Matrices of a short side up to
128 are always multiplied as with ``"split"``.)  Long inner products add the rounding of their sums: a sum over ``l`` terms
is made of 3 l / 32 additions to one fp32 accumulator (three products of 32 terms each), every one off by at most
2^-24 of the sum of squares that is on the Gram matrix's diagonal, so A is off by 3 l / 32 * 2^-24 of itself at most, and
b x^3 + c x^5 by no more than that (its derivative in A is under 1 from x = 0.6 to 1.2).
"""
from __future__ import annotations

import gc
import math

import pytest
import torch

import _matrix_oracle as M
from fairscale_amd.optim import Adam, GradScaler, Muon, Precision, clip_grad_norm_, grad_pass, momentum_pass, orthogonalize

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
PRODUCT_ERROR = {"half": 2 * 1.9e-3, "split": 2 * 2.6e-6}


def default_products(dtype):
    return "half" if dtype == torch.bfloat16 else "split"


def tolerance(dtype, products, longest=0):
    return torch.finfo(dtype).eps / 2 + PRODUCT_ERROR[products] + 3 * longest / 32 * 2**-24


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(n * (k + 3) for k, n in enumerate(shape)))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def check_orth(matrices, results, products=None, factor=1.0, **how):
    for u, o in zip(matrices, results):
        assert o.shape == u.shape and o.dtype == u.dtype
        want = M.orthogonal(u, **how)
        flat_o, flat_w = o.reshape(-1, *o.shape[-2:]), want.reshape(-1, *want.shape[-2:])
        for x, y in zip(flat_o, flat_w):
            assert M.relative(x, y) <= factor * tolerance(u.dtype, products or default_products(u.dtype), max(u.shape[-2:])), (tuple(u.shape), u.dtype)


# ---- orthogonalize ------------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 2), (2, 1), (1, 300), (300, 1), (3, 5), (16, 16), (63, 64), (64, 65), (65, 63), (64, 64), (127, 129), (128, 128), (129, 128), (130, 257),
          (200, 64), (64, 1000), (1000, 64), (255, 256), (257, 255), (300, 700), (700, 300), (512, 512), (640, 385)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_one_matrix(shape, dtype):
    u = randn(*shape, dtype=dtype)
    keep = u.clone()
    check_orth([u], orthogonalize([u]))
    assert torch.equal(u, keep)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("products", ["half", "split"])
def test_a_list_of_all_shapes_in_one_call(dtype, products):
    us = [randn(*s, dtype=dtype, seed=1) for s in SHAPES]
    check_orth(us, orthogonalize(us, products=products), products)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_larger_matrices(dtype):
    us = [randn(1111, 2050, dtype=dtype), randn(1536, 700, dtype=dtype), randn(1, 20000, dtype=dtype), randn(40, 9001, dtype=dtype)]
    check_orth(us, orthogonalize(us))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_batches_are_matrices_of_their_own(dtype):
    u = randn(5, 48, 130, dtype=dtype) * torch.tensor([1.0, 1e-2, 30.0, 1.0, 5.0], device="cuda", dtype=dtype).view(5, 1, 1)
    v = randn(2, 3, 70, 33, dtype=dtype)
    got = orthogonalize([u, v])
    check_orth([u, v], got)
    for k in range(5):
        assert torch.equal(got[0][k], orthogonalize([u[k]])[0]), "a matrix gives the same bits alone and in a batch"


@pytest.mark.parametrize("kind", ["low_rank", "decay"])
@pytest.mark.parametrize("dtype, products", [(torch.float32, "split"), (torch.float32, "half"), (torch.bfloat16, "half"), (torch.float16, "split")], ids=str)
def test_matrices_far_from_orthogonal(kind, dtype, products):
    """Directions four orders apart: the first iterate's rounding is what grows most here."""
    s, l = 256, 512
    if kind == "low_rank":
        u = randn(s, 8) @ randn(8, l) + 0.01 * randn(s, l)
    else:
        q1, q2 = torch.linalg.qr(randn(s, s).cpu())[0], torch.linalg.qr(randn(l, s).cpu())[0]
        u = ((q1 * torch.logspace(0, -4, s)) @ q2.t()).cuda()
    u = u.to(dtype)
    allowed = torch.finfo(dtype).eps / 2 + (2 * 1.9e-3 if products == "half" else 2 * 3e-5)
    assert M.relative(orthogonalize([u], products=products)[0], M.orthogonal(u)) <= allowed


def test_views_are_read_and_written_where_they_lie():
    base = randn(3, 90, 150)
    views = [base[0], base[0].t(), base[1, 5:80, 7:130], base[1, 5:80, 7:130].t(), base.transpose(1, 2), base[:, 3:4], base[:, :, 4:5], base[2, 10:11], base[2, :, 9:10]]
    check_orth(views, orthogonalize(views))
    into = torch.full((3, 90, 150), 7.0, device="cuda")
    outs = [into[1, 5:80, 7:130], into[2, :40, :60].t()]
    us = [randn(75, 123), randn(40, 60, seed=3).t()]
    got = orthogonalize(us, out=outs)
    assert got[0] is outs[0]
    check_orth(us, got)
    mask = torch.ones_like(into, dtype=torch.bool)
    mask[1, 5:80, 7:130] = False
    mask[2, :40, :60] = False
    assert (into[mask] == 7.0).all(), "what lies around the results is left as it was"


def test_results_over_the_matrices():
    us = [randn(70, 30), randn(4, 33, 65)]
    keep = [u.clone() for u in us]
    got = orthogonalize(us, out=us)
    assert all(a is b for a, b in zip(got, us))
    check_orth(keep, us)


def test_empty_matrices_and_lists():
    assert orthogonalize([]) == []
    got = orthogonalize([torch.zeros(0, 5, device="cuda"), randn(4, 9), torch.zeros(3, 0, device="cuda"), torch.zeros(0, 4, 4, device="cuda")])
    assert [tuple(o.shape) for o in got] == [(0, 5), (4, 9), (3, 0), (0, 4, 4)]
    check_orth([randn(4, 9)], [got[1]])
    assert orthogonalize([torch.zeros(0, 5, device="cuda")])[0].shape == (0, 5)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_zeros_stay_zeros_and_values_that_are_not_finite_stay_in_their_matrix(dtype):
    us = [torch.zeros(70, 130, device="cuda", dtype=dtype), randn(70, 130, dtype=dtype), randn(3, 70, 130, dtype=dtype), randn(70, 130, dtype=dtype)]
    us[2][1, 69, 129] = math.inf
    us[3][0, 0] = math.nan
    got = orthogonalize(us)
    assert (got[0] == 0).all()
    check_orth([us[1], us[2][0], us[2][2]], [got[1], got[2][0], got[2][2]])
    assert got[2][1].isnan().all() and got[3].isnan().all()


@pytest.mark.parametrize("dtype, scale", [(torch.float32, 1e-38), (torch.float32, 1e37), (torch.float32, 1e-30), (torch.float16, 6e-8), (torch.float16, 3e4),
                                          (torch.bfloat16, 1e-38), (torch.bfloat16, 1e37)], ids=str)
def test_very_small_and_very_large_matrices(dtype, scale):
    sign = torch.where(randn(60, 100) > 0, 1.0, -1.0)
    u = (sign * scale).to(dtype)
    check_orth([u], orthogonalize([u], eps=1e-45 if scale < 1e-20 else 1e-7), eps=1.4e-45 if scale < 1e-20 else 1e-7)
    if scale < 1e-20:
        # Far under eps the exact result is 3.4445^5 U / eps < 1e-20.  X0 is held in steps of 2^-39 (halves of 2^-24 times 2^-15),
        # so an entry is off by at most 2^-40, which five steps multiply by at most 3.4445 each.
        got, want = orthogonalize([u])[0], M.orthogonal(u)
        assert (got.double().cpu() - want).norm().item() <= 3.4445**5 * 2**-40 * math.sqrt(u.numel())


@pytest.mark.parametrize("coefficients, steps", [((1.5, -0.5, 0.0), 8), ((1.875, -1.25, 0.375), 6), ((0.0, 0.0, 0.0), 2), ((-3.4445, 4.7750, -2.0315), 3),
                                                 ((1.0, 0.0, 0.0), 1), ((2.0, -1.5, 0.5), 12), ((8.0, 0.0, 0.0), 3), (M.COEFFICIENTS, 1), (M.COEFFICIENTS, 2), (M.COEFFICIENTS, 10)])
def test_other_steps_and_coefficients(coefficients, steps):
    u = randn(90, 140)
    got = orthogonalize([u], steps=steps, coefficients=coefficients)[0]
    # twelve steps and ten may add the errors of so many products
    assert M.relative(got, M.orthogonal(u, steps, coefficients)) <= max(1, steps / 5) * tolerance(torch.float32, "split")


def test_singular_values_come_near_one():
    u = randn(300, 500)
    s = torch.linalg.svdvals(orthogonalize([u])[0].double().cpu())
    assert s.max() < 1.21 and s.min() > 0.3


def test_scale_of_the_matrix_does_not_matter():
    u = randn(100, 200)
    a, b = orthogonalize([u, u * 1024.0])
    assert torch.equal(a, b), "powers of two leave the bits alone"


def test_list_longer_than_a_table_and_chunks():
    us = [randn(8 + k % 5, 70 - k, seed=k) for k in range(53)]
    check_orth(us, orthogonalize(us))


def test_list_that_needs_several_chunks():
    """Ten matrices of 0.55 GB of intermediates: more than one chunk's 4 GiB."""
    base = randn(2, 4096, 4096, dtype=torch.bfloat16)
    us = [base[k % 2] for k in range(5)] + [base[0].expand(5, 4096, 4096)]
    got = orthogonalize(us, products="split")
    one = orthogonalize([base[0], base[1]], products="split")
    for k in range(5):
        assert torch.equal(got[k], one[k % 2])
    assert all(torch.equal(got[5][k], one[0]) for k in range(5))


# ---- momentum -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("grad_type", TYPES, ids=str)
@pytest.mark.parametrize("update_type", TYPES, ids=str)
@pytest.mark.parametrize("nesterov", [True, False])
def test_momentum_pass(grad_type, update_type, nesterov):
    shapes = [(1,), (7,), (0,), (8191,), (8192,), (8193,), (3, 5, 7), (100, 333), (20001,)]
    grads = [randn(*s, dtype=grad_type, scale=4.0) if math.prod(s) else torch.zeros(s, device="cuda", dtype=grad_type) for s in shapes]
    bufs = [randn(*s, seed=1, scale=1e-2) if math.prod(s) else torch.zeros(s, device="cuda") for s in shapes]
    before = [b.clone() for b in bufs]
    updates = [torch.empty(s, device="cuda", dtype=update_type) for s in shapes]
    got = momentum_pass(grads, bufs, 0.95, nesterov=nesterov, scale=64.0, updates=updates)
    assert got.updates is updates or all(a is b for a, b in zip(got.updates, updates))
    assert got.found_inf.item() == 0.0 and got.norms.shape == (len(shapes),) and got.norms.dtype == torch.float32
    for k, (g, b, u) in enumerate(zip(grads, before, updates)):
        m, want = M.momentum(g, b, 0.95, nesterov, 64.0)
        # five roundings of fp32 at the size of the larger operand
        atol = 5 * 2**-24 * (g.double().abs().max().item() / 64 + b.abs().max().item()) if g.numel() else 0.0
        assert ((bufs[k].double().cpu() - m).abs() <= atol).all()
        half_step = torch.finfo(update_type).eps / 2
        tiny = torch.finfo(update_type).smallest_normal * half_step  # a subnormal's rounding
        assert ((u.double().cpu() - want).abs() <= want.abs() * half_step + 2 * atol + tiny).all()
        norm = u.double().norm().item()
        assert abs(got.norms[k].item() - norm) <= norm * 2**-23


def test_momentum_updates_default_to_the_gradients_type_and_may_lie_over_them():
    g, m = randn(50, 60, dtype=torch.bfloat16), torch.zeros(50, 60, device="cuda")
    first = momentum_pass([g], [m]).updates[0]
    assert first.dtype == torch.bfloat16 and first.data_ptr() != g.data_ptr()
    m.zero_()
    momentum_pass([g], [m], updates=[g])
    assert torch.equal(g, first)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_momentum_of_views_that_start_anywhere(offset):
    n = 30011
    g = randn(n + offset, dtype=torch.float16)[offset:]
    flat = randn(n + 8)
    m, far = flat[8 - offset:n + 8 - offset], flat.clone()
    u = torch.zeros(n + 16, device="cuda", dtype=torch.bfloat16)
    want_m, want = M.momentum(g, m, 0.9, True)
    momentum_pass([g], [m], 0.9, updates=[u[offset:n + offset]])
    assert M.relative(m, want_m) < 2**-22 and M.relative(u[offset:n + offset], want) < 2**-8
    assert (u[:offset] == 0).all() and (u[n + offset:] == 0).all() and torch.equal(flat[:8 - offset], far[:8 - offset]) and torch.equal(flat[n + 8 - offset:], far[n + 8 - offset:])


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_momentum_raises_the_flag_for_what_is_not_finite(bad):
    grads, bufs = [randn(100), randn(9000, dtype=torch.float32)], [torch.zeros(100, device="cuda"), torch.zeros(9000, device="cuda")]
    grads[1][8999] = bad
    flag = torch.zeros(1, device="cuda")
    got = momentum_pass(grads, bufs, found_inf=flag)
    assert got.found_inf is flag and flag.item() == 1.0
    assert got.norms[0].isfinite() and not got.norms[1].isfinite()
    clean = momentum_pass([grads[0]], [bufs[0]], found_inf=flag)
    assert clean.found_inf.item() == 1.0, "never cleared"


def test_momentum_flags_an_update_that_its_type_cannot_hold():
    g, m = torch.full((10,), 1e6, device="cuda"), torch.zeros(10, device="cuda")
    assert momentum_pass([g], [m], 0.0, updates=[torch.empty(10, device="cuda", dtype=torch.float16)]).found_inf.item() == 1.0
    assert momentum_pass([g], [m], 0.0).found_inf.item() == 0.0
    big = torch.full((10,), 3e38, device="cuda")  # its sum of squares is far over fp32
    assert momentum_pass([big], [torch.zeros(10, device="cuda")], 0.0).found_inf.item() == 0.0


def test_momentum_scale_may_be_a_tensor():
    g, a, b = randn(300, dtype=torch.float16), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    momentum_pass([g], [a], scale=3.0)
    momentum_pass([g], [b], scale=torch.tensor([3.0], device="cuda"))
    assert torch.equal(a, b)


def test_momentum_list_longer_than_a_table():
    grads, bufs = [randn(1 + 13 * k) for k in range(150)], [torch.zeros(1 + 13 * k, device="cuda") for k in range(150)]
    got = momentum_pass(grads, bufs, 0.5, nesterov=False)
    for g, m, u in zip(grads, bufs, got.updates):
        assert torch.equal(m, g * 0.5) and torch.equal(u, m)


# ---- refusals -----------------------------------------------------------------------------------------------------

def test_refusals():
    a, h = randn(8, 8), randn(8, 8, dtype=torch.float16)
    for call in (lambda: orthogonalize([a, h]), lambda: orthogonalize([a[:, ::2]]), lambda: orthogonalize([a[0]]), lambda: orthogonalize([a.to_sparse()]),
                 lambda: orthogonalize([a], out=[h]), lambda: orthogonalize([a], out=[a[:4]]), lambda: orthogonalize([a], out=[torch.empty(8, 8, device="cuda").t()]),
                 lambda: orthogonalize([a], out=[]), lambda: orthogonalize([a, a], out=[a, a]), lambda: orthogonalize([a, a.cpu()]),
                 lambda: orthogonalize([a], out=[torch.empty(1, 8, device="cuda").expand(8, 8)]),
                 lambda: momentum_pass([a], [h]), lambda: momentum_pass([a, h], [a, a]), lambda: momentum_pass([a], [a[:4]]), lambda: momentum_pass([a.t()], [a]),
                 lambda: momentum_pass([a, a], [h.float(), h.float()], updates=[a, a]), lambda: momentum_pass([a, a.clone()], [a, a]),
                 lambda: momentum_pass([a], [a.clone()], scale=torch.ones(2, device="cuda")), lambda: momentum_pass([a], [a.clone()], scale=torch.ones(1)),
                 lambda: momentum_pass([a], [a.clone()], scale=0.0), lambda: momentum_pass([a], [a.clone()], 1.0),
                 lambda: momentum_pass([a], [a.clone()], found_inf=torch.zeros(1)), lambda: momentum_pass([a], [a.clone()], updates=[a.double()])):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: orthogonalize([a], products="tf32"), lambda: orthogonalize([a], coefficients=(1.0,)), lambda: orthogonalize([a], steps=1.5)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        orthogonalize([a], steps=0)


# ---- Muon ---------------------------------------------------------------------------------------------------------

MODES = [("full", Precision.FULL_PRECISION, torch.float32), ("mixed16", Precision.MIXED_PRECISION, torch.float16), ("mixedb", Precision.MIXED_PRECISION, torch.bfloat16),
         ("mem16", Precision.MEMORY_EFFICIENT_MIXED_PRECISION, torch.float16), ("memb", Precision.MEMORY_EFFICIENT_MIXED_PRECISION, torch.bfloat16)]


def close_step(got, want, before, dtype, products, lr, ratio, cols_rows):
    """Parameter after a step: the rounding of its type, three of fp32, and lr * ratio times the error of the orthogonalised update."""
    norm = lr * ratio * math.sqrt(min(cols_rows)) * 1.21  # of lr * ratio * O: singular values are at most 1.21
    allowed = (torch.finfo(dtype).eps / 2 + 3 * 2**-24) * want.norm().item() + norm * (tolerance(torch.float32, products))
    assert (got.double().cpu() - want).norm().item() <= allowed


@pytest.mark.parametrize("name, precision, dtype", MODES, ids=[m[0] for m in MODES])
@pytest.mark.parametrize("how, nesterov", [(None, True), ("match_rms_adamw", False)])
def test_muon_steps(name, precision, dtype, how, nesterov):
    shapes = [(30, 50), (50, 30), (1, 9), (129, 64), (3, 20, 40), (2, 2, 40, 20), (256, 300)]
    lr, scale = 0.05, 8.0
    params = [torch.nn.Parameter(randn(*s, dtype=dtype, scale=0.1)) for s in shapes]
    opt = Muon(params, lr=lr, nesterov=nesterov, adjust_lr_fn=how, precision=precision)
    buffers = [torch.zeros(s, dtype=torch.float64) for s in shapes]
    for n in range(3):
        masters = opt.fp32_param_groups[0]["params"] if opt.mixed_precision else params
        before = [w.detach().double().cpu() for w in masters]
        for k, p in enumerate(params):
            p.grad = randn(*p.shape, seed=10 + n, dtype=dtype)
            if "momentum_buffer" in opt.state[p]:
                buffers[k] = opt.state[p]["momentum_buffer"].double().cpu()
        opt.step(scale=scale)
        for k, p in enumerate(params):
            want, m = M.step(before[k], p.grad, buffers[k], lr=lr, nesterov=nesterov, scale=scale, how=how)
            assert M.relative(opt.state[p]["momentum_buffer"], m) <= 4 * 2**-24
            for x, y, b in zip(masters[k].reshape(-1, *p.shape[-2:]), want.reshape(-1, *p.shape[-2:]), before[k].reshape(-1, *p.shape[-2:])):
                close_step(x, y, b, masters[k].dtype, opt.products, lr, M.ratio(*p.shape[-2:], how), p.shape[-2:])
            if opt.mixed_precision:
                assert torch.equal(p.detach(), masters[k].to(dtype)), "the copy is the rounded master"


def test_muon_groups_row_blocks_and_parameters_without_gradients():
    qkv, w, idle = (torch.nn.Parameter(randn(96, 40)), torch.nn.Parameter(randn(20, 30)), torch.nn.Parameter(randn(5, 5)))
    keep = idle.detach().clone()
    opt = Muon([{"params": [qkv], "row_blocks": 3, "lr": 0.1}, {"params": [w, idle], "weight_decay": 0.0, "ns_steps": 3}], lr=0.02)
    before = [qkv.detach().double().cpu(), w.detach().double().cpu()]
    qkv.grad, w.grad = randn(96, 40, seed=5), randn(20, 30, seed=6)
    opt.step()
    want, _ = M.step(before[0], qkv.grad, torch.zeros(96, 40), lr=0.1, row_blocks=3)
    assert M.relative(qkv, want) < 1e-5
    want, _ = M.step(before[1], w.grad, torch.zeros(20, 30), lr=0.02, weight_decay=0.0, steps=3)
    assert M.relative(w, want) < 1e-5
    assert torch.equal(idle.detach(), keep) and idle not in opt.state


def test_muon_is_momentum_pass_then_orthogonalize():
    """The fused step and the operators it is made of, used together, give the same momentum bit for bit and the same parameters."""
    p = torch.nn.Parameter(randn(130, 200))
    p.grad = randn(130, 200, seed=2)
    w, m = p.detach().clone(), torch.zeros(130, 200, device="cuda")
    opt = Muon([p], lr=0.1, weight_decay=0.01)
    for _ in range(3):
        opt.step(scale=2.0)
        stats = momentum_pass([p.grad], [m], 0.95, scale=2.0)
        w = w * (1 - 0.1 * 0.01) - 0.1 * orthogonalize(stats.updates)[0]
        assert torch.equal(opt.state[p]["momentum_buffer"], m)
        assert M.relative(p, w) < 1e-6


def test_muon_with_scaler_clipping_and_adam_beside_it():
    """As a training program has them: one scaler and one clip over the gradients of both optimizers."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(40, 70), torch.nn.Tanh(), torch.nn.Linear(70, 8)).cuda()
    matrices, rest = [p for p in model.parameters() if p.dim() == 2], [p for p in model.parameters() if p.dim() < 2]
    muon, adam = Muon(matrices, lr=0.02), Adam(rest, lr=1e-2)
    scaler = GradScaler("cuda", init_scale=256.0)
    x, y = randn(64, 40), randn(64, 8, seed=1)
    for _ in range(3):
        with torch.autocast("cuda", dtype=torch.float16):
            loss = (model(x) - y).square().mean()
        scaler.scale(loss).backward()
        scaler.unscale_(muon)
        scaler.unscale_(adam)
        norm, factor = clip_grad_norm_(list(model.parameters()), 0.1, fold="device")
        before = [(p.detach().double().cpu(), muon.state[p]["momentum_buffer"].double().cpu() if p in muon.state else torch.zeros(p.shape)) for p in matrices]
        muon.step(scale=factor)
        adam.step(scale=factor)
        for p, (w, m) in zip(matrices, before):
            want, m2 = M.step(w, p.grad, m, lr=0.02, scale=factor.item())
            assert M.relative(p, want) < 1e-5 and M.relative(muon.state[p]["momentum_buffer"], m2) < 1e-6
        scaler.update()
        muon.zero_grad()
        adam.zero_grad()


def test_muon_resumes_bit_for_bit():
    for name, precision, dtype in MODES:
        p = torch.nn.Parameter(randn(40, 60, dtype=dtype))
        opt = Muon([p], precision=precision)
        p.grad = randn(40, 60, seed=1, dtype=dtype)
        opt.step()
        q = torch.nn.Parameter(p.detach().clone())
        other = Muon([q], precision=precision)
        other.load_state_dict(opt.state_dict())
        q.grad = p.grad.clone()
        opt.step()
        other.step()
        assert torch.equal(p.detach(), q.detach()), name
        assert torch.equal(opt.state[p]["momentum_buffer"], other.state[q]["momentum_buffer"]), name


def test_muon_refusals_change_nothing():
    p, q = torch.nn.Parameter(randn(20, 30)), torch.nn.Parameter(randn(8, 8))
    opt = Muon([{"params": [p]}, {"params": [q]}])
    p.grad, q.grad = randn(20, 30, seed=1), randn(8, 8, seed=1)
    opt.step()
    keep = [t.detach().clone() for t in (p, q, opt.state[p]["momentum_buffer"], opt.state[q]["momentum_buffer"])]

    def unchanged():
        assert all(torch.equal(a, b.detach()) for a, b in zip(keep, (p, q, opt.state[p]["momentum_buffer"], opt.state[q]["momentum_buffer"])))

    for scale in (torch.ones(2, device="cuda"), torch.ones(1), torch.ones(1, device="cuda", dtype=torch.float16)):
        with pytest.raises(RuntimeError):
            opt.step(scale=scale)
        unchanged()
    for scale in (0.0, math.inf, math.nan):
        with pytest.raises(RuntimeError):
            opt.step(scale=scale)
        unchanged()
    good = opt.state[q]["momentum_buffer"]
    for bad in (good.half(), good[:4], good.cpu(), opt.state[p]["momentum_buffer"]):
        opt.state[q]["momentum_buffer"] = bad
        with pytest.raises(RuntimeError):
            opt.step()
        opt.state[q]["momentum_buffer"] = good
        unchanged()
    q.grad = randn(8, 8, seed=1).t()
    with pytest.raises(RuntimeError):
        opt.step()
    unchanged()


def test_muon_gradient_that_is_not_finite_stays_with_its_matrix():
    p, q = torch.nn.Parameter(randn(20, 30)), torch.nn.Parameter(randn(2, 20, 30))
    opt = Muon([p, q])
    p.grad, q.grad = randn(20, 30, seed=1), randn(2, 20, 30, seed=1)
    q.grad[1, 3, 4] = math.inf
    opt.step()
    assert p.isfinite().all() and q[0].isfinite().all() and q[1].isnan().all()


# ---- streams, graphs ----------------------------------------------------------------------------------------------

def test_calls_on_two_streams_at_once():
    us = [randn(300, 500, seed=k) for k in range(4)]
    want = [orthogonalize([u])[0] for u in us]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None] * 4
    for _ in range(3):
        for k, u in enumerate(us):
            with torch.cuda.stream(streams[k % 2]):
                got[k] = orthogonalize([u])[0]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_orthogonalize_and_momentum_in_a_replayed_graph():
    u, g, m = randn(200, 90), randn(200, 90, dtype=torch.float16), torch.zeros(200, 90, device="cuda")
    orthogonalize([u])
    momentum_pass([g], [m.clone()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stats = momentum_pass([g], [m])
        o = orthogonalize([u])[0]
    eager_m = torch.zeros_like(m)
    for n in range(4):
        u.copy_(randn(200, 90, seed=n))
        g.copy_(randn(200, 90, seed=n + 10, dtype=torch.float16))
        graph.replay()
        torch.cuda.synchronize()
        want = momentum_pass([g], [eager_m])
        assert torch.equal(o, orthogonalize([u])[0]) and torch.equal(m, eager_m) and torch.equal(stats.updates[0], want.updates[0])
        assert torch.equal(stats.norms, want.norms) and stats.found_inf.item() == 0.0


def test_two_graphs_share_nothing():
    a, b = randn(100, 150), randn(64, 300)
    want = orthogonalize([a]), orthogonalize([b])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for u in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(orthogonalize([u])[0])
        graphs.append(graph)
    s = torch.cuda.Stream()
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(s):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0][0]) and torch.equal(outs[1], want[1][0])


def test_muon_step_in_a_replayed_graph():
    p, q = torch.nn.Parameter(randn(60, 80)), torch.nn.Parameter(randn(60, 80))
    p.grad, q.grad = randn(60, 80, seed=1), randn(60, 80, seed=1)
    opt, eager = Muon([p]), Muon([q])
    graph = torch.cuda.CUDAGraph()
    opt.step()
    eager.step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for n in range(3):
        p.grad.copy_(randn(60, 80, seed=n + 2))
        q.grad.copy_(p.grad)
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        assert torch.equal(p.detach(), q.detach())


def test_muon_refuses_to_make_its_momentum_inside_a_capture():
    p = torch.nn.Parameter(randn(8, 8))
    p.grad = randn(8, 8, seed=1)
    opt = Muon([p])
    keep = p.detach().clone()
    spare = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        spare.add_(1.0)
        with pytest.raises(RuntimeError, match="capture"):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), keep)


def test_same_inputs_give_the_same_bits():
    us = [randn(500, 300), randn(7, 64, 200)]
    first = orthogonalize(us)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, orthogonalize(us)))
    gc.collect()


@pytest.mark.parametrize("products", ["half", "split"])
@pytest.mark.parametrize("others", [[(1100, 1024)] * 30, [(4096, 2048)] * 12, [(5, 7)]], ids=["30_of_1100", "12_of_4096", "small"])
def test_what_a_matrix_gives_does_not_depend_on_the_list(products, others):
    """The list decides the tiles (64, 128 or 256) of every launch, and so which of them run into the ends of the matrix."""
    us = [randn(700, 900), randn(901, 640), randn(333, 2049), randn(130, 4100), randn(64, 256), randn(200, 130), randn(2, 310, 515)]
    alone = [orthogonalize([u], products=products)[0] for u in us]
    rest = [randn(*others[0], seed=9)] * len(others)
    for k, (a, b) in enumerate(zip(alone, orthogonalize(us + rest, products=products))):
        assert torch.equal(a, b), us[k].shape
    check_orth(us, alone, products)


def test_momentum_pass_over_empty_tensors_only():
    got = momentum_pass([torch.zeros(0, device="cuda"), torch.zeros(3, 0, device="cuda")], [torch.zeros(0, device="cuda"), torch.zeros(3, 0, device="cuda")])
    assert got.found_inf.item() == 0.0 and (got.norms == 0).all()


# ---- memory shared between the tensors of a call -------------------------------------------------------------------

@pytest.mark.parametrize("rows", [90, 300])
def test_halves_of_the_columns_of_one_tensor_in_place(rows):
    whole = randn(rows, 400, seed=3)
    left, right = whole[:, :160], whole[:, 160:]
    want = [t.clone() for t in orthogonalize([left, right])]
    orthogonalize([left, right], out=[left, right])
    assert torch.equal(left, want[0]) and torch.equal(right, want[1])


@pytest.mark.parametrize("rows", [20, 300])
def test_calls_whose_results_share_memory_are_refused_and_change_nothing(rows):
    a, b, g = randn(rows, 320, seed=1), randn(rows, 320, seed=2), randn(rows, 320, seed=3)
    flat = torch.zeros(rows * 320 + 8, device="cuda")
    shifted = [flat[:rows * 320].view(rows, 320), flat[4:4 + rows * 320].view(rows, 320)]
    keep = [t.clone() for t in (a, b, g, flat)]
    for call in (lambda: orthogonalize([a, b], out=[b, a]), lambda: orthogonalize([a, b], out=[a, a]), lambda: orthogonalize([a, b], out=shifted),
                 lambda: orthogonalize([shifted[0]], out=[shifted[1]]), lambda: momentum_pass([g], [a], updates=[a]),
                 lambda: momentum_pass([g, b], [a, b]), lambda: momentum_pass([g, b], [a, randn(rows, 320)], updates=[b, g]),
                 lambda: momentum_pass([g, b], shifted), lambda: momentum_pass([shifted[0]], [shifted[1]])):
        with pytest.raises(RuntimeError, match="share"):
            call()
    p = [torch.nn.Parameter(t) for t in shifted]
    for q in p:
        q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="share"):
        Muon(p).step()
    assert all(torch.equal(t, k) for t, k in zip((a, b, g, flat), keep))


def test_parameters_in_one_buffer():
    flat = randn(2 * 300 * 200, seed=5)
    apart = [torch.nn.Parameter(t.clone()) for t in flat.view(2, 300, 200)]
    together = [torch.nn.Parameter(t) for t in flat.view(2, 300, 200)]
    for ps in (apart, together):
        for k, p in enumerate(ps):
            p.grad = randn(300, 200, seed=6 + k)
        Muon(ps, lr=0.1).step()
    assert torch.equal(flat.view(2, 300, 200), torch.stack([p.detach() for p in apart]))


# ---- sizes -----------------------------------------------------------------------------------------------------------

def test_lists_of_several_thousand_rows():
    """Every matrix of a long list is found: more rows than a wave looks at once, and more than 64 times as many."""
    shapes = [(3, 5), (150, 140), (1, 1), (0, 4)]
    us = [randn(*shapes[k % 4], seed=k % 12) for k in range(4500)]
    alone = {k: orthogonalize([us[k]])[0] for k in range(12)}
    got = orthogonalize(us)
    assert all(torch.equal(o, alone[k % 12]) for k, o in enumerate(got))
    stats = momentum_pass(us, [torch.zeros_like(u) for u in us], 0.5, nesterov=False)
    want = [momentum_pass([us[k]], [torch.zeros_like(us[k])], 0.5, nesterov=False) for k in range(12)]
    assert all(torch.equal(u, want[k % 12].updates[0]) for k, u in enumerate(stats.updates))
    assert torch.equal(stats.norms, torch.cat([w.norms for w in want]).repeat(375))


@pytest.mark.parametrize("tall", [False, True])
def test_matrix_of_more_than_2_31_elements(tall):
    """Entries only at (i, 2 i): the singular values are their sizes, so the result has the polynomial's values there and zeros elsewhere."""
    s, l = 32800, 65600
    d = torch.full((s,), 0.25, device="cuda")
    d[:3], d[-3:], d[s // 2] = 300.0, -200.0, 250.0
    u = torch.zeros((l, s) if tall else (s, l), dtype=torch.bfloat16, device="cuda")
    at = lambda t: t.as_strided((s,), (2 * s + 1,) if tall else (l + 2,))
    at(u).copy_(d)
    out = orthogonalize([u], steps=1)[0]
    x = d.double() / d.double().norm()
    want = 3.4445 * x - 4.7750 * x**3 + 2.0315 * x**5
    got = at(out).double()
    # 11 bits of A, B and X in the products and 8 in the result: (|b| x^3 * 3 + |c| x^5 * 5) 2^-11 + |result| 2^-8, and an fp32 sum's 2^-20
    bound = (3 * 4.7750 * x.abs()**3 + 5 * 2.0315 * x.abs()**5) * 2.0**-11 + want.abs() * (2.0**-8 + 2.0**-20) + 1e-9
    assert ((got - want).abs() <= bound).all()
    at(out).zero_()
    assert int(torch.count_nonzero(out)) == 0


# ---- states that are assigned, as a sharded optimizer's resume does --------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_muon_resumes_from_an_assigned_state(dtype):
    """``optimizer.state[p] = {...}`` in a new program, then steps, a checkpoint and another resume: each bit as in the program that went on."""
    p = torch.nn.Parameter(randn(40, 60, dtype=dtype))
    opt = Muon([p])
    grads = [randn(40, 60, seed=k + 1, dtype=dtype) for k in range(4)]
    for k in range(2):
        p.grad = grads[k].clone()
        opt.step()
    for resume in range(2):
        q = torch.nn.Parameter(torch.zeros_like(p))  # the masters alone carry the values
        other = Muon([q])
        other.state[q] = {key: value.clone() for key, value in opt.state_dict()["state"][0].items()}
        for o, w in ((opt, p), (other, q)):
            w.grad = grads[2 + resume].clone()
            o.step()
        assert torch.equal(p.detach(), q.detach())
        saved, kept = other.state_dict()["state"][0], opt.state_dict()["state"][0]
        assert torch.equal(saved["master"], kept["master"]) and torch.equal(saved["momentum_buffer"], kept["momentum_buffer"])
        assert torch.equal(saved["master"].to(dtype), q.detach())
        p, opt = q, other


def test_muon_refuses_masters_it_cannot_step_and_changes_nothing():
    p = torch.nn.Parameter(randn(20, 30, dtype=torch.bfloat16))
    opt = Muon([p])
    p.grad = randn(20, 30, seed=1, dtype=torch.bfloat16)
    opt.step()
    keep, momentum, good = p.detach().clone(), opt.state[p]["momentum_buffer"].clone(), opt.state[p]["master"]
    for bad in (good.half(), good[:4], good.cpu(), torch.zeros(30, 20, device="cuda").t(), opt.state[p]["momentum_buffer"]):
        opt.state[p]["master"] = bad
        with pytest.raises(RuntimeError):
            opt.step()
        assert torch.equal(p.detach(), keep) and torch.equal(opt.state[p]["momentum_buffer"], momentum)


def test_muon_refuses_to_make_a_master_inside_a_capture():
    p = torch.nn.Parameter(randn(8, 8, dtype=torch.float16))
    p.grad = randn(8, 8, seed=1, dtype=torch.float16)
    opt = Muon([p])
    opt.step()
    keep = p.detach().clone()
    opt.state[p] = {"momentum_buffer": opt.state[p]["momentum_buffer"]}
    spare = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        spare.add_(1.0)
        with pytest.raises(RuntimeError, match="capture"):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), keep)


# ---- groups ------------------------------------------------------------------------------------------------------------

def test_muon_refuses_a_group_before_another_one_is_stepped():
    """The second group's matrix has more rows than a call takes: the first group stays as it was."""
    p, q = torch.nn.Parameter(randn(20, 30)), torch.nn.Parameter(torch.zeros((1 << 20) + 1, 1, device="cuda"))
    p.grad, q.grad = randn(20, 30, seed=1), torch.ones_like(q)
    keep = p.detach().clone()
    opt = Muon([{"params": [p]}, {"params": [q]}])
    for _ in range(2):
        with pytest.raises(RuntimeError, match="2\\^20"):
            opt.step()
        assert torch.equal(p.detach(), keep) and (opt.state[p]["momentum_buffer"] == 0).all() and (q == 0).all()
    q.grad = None
    opt.step()
    alone = torch.nn.Parameter(keep.clone())
    alone.grad = p.grad
    Muon([alone]).step()
    assert torch.equal(p, alone)


def test_muon_groups_of_different_sizes_share_a_workspace():
    """Each bit as from an optimizer of its own: large before small, small before large, one that needs no workspace."""
    shapes = [(300, 200), (700, 900), (40, 50), (150, 4000)]
    ps, qs = ([torch.nn.Parameter(randn(*s)) for s in shapes] for _ in range(2))
    for k, (p, q) in enumerate(zip(ps, qs)):
        p.grad, q.grad = randn(*shapes[k], seed=k + 1), randn(*shapes[k], seed=k + 1)
    opt = Muon([{"params": [p], "ns_steps": 5 - k % 2} for k, p in enumerate(ps)])
    apart = [Muon([q], ns_steps=5 - k % 2) for k, q in enumerate(qs)]
    for _ in range(3):
        opt.step()
        for o in apart:
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_muon_of_a_convolutions_weight():
    """As the documentation says: a leaf of two dimensions over the weight's memory, which is given the weight's gradient before a step."""
    conv = torch.nn.Conv2d(5, 12, 3).cuda()
    flat = torch.nn.Parameter(conv.weight.detach().view(12, -1))
    opt = Muon([flat], lr=0.1)
    conv(randn(2, 5, 8, 8)).square().mean().backward()
    before = conv.weight.detach().double().cpu().view(12, -1)
    flat.grad = conv.weight.grad.view(12, -1)
    opt.step()
    want, _ = M.step(before, flat.grad, torch.zeros(12, 45), lr=0.1)
    assert M.relative(conv.weight.view(12, -1), want) < 1e-5
    with pytest.raises(ValueError, match="non-leaf"):
        Muon([conv.weight.view(12, -1)])
