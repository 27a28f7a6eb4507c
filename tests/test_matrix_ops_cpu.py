"""What the matrix operators say without a GPU: their C entries refuse bad arguments before they touch a device, the workspace
sizes are those of the documented storage, and the Python layer names what it will not take."""
from __future__ import annotations

import copy
import ctypes
import math
import pickle

import pytest
import torch

from fairscale_amd import _cabi, matrix_ops
from fairscale_amd.optim import Muon, Precision, momentum_pass, orthogonalize
import _matrix_oracle as M

L = _cabi.lib()
FAKE = 1 << 20  # an address nothing is read from


def options(steps=5, coefficients=M.COEFFICIENTS, eps=1e-7, products=_cabi.PRODUCTS_HALF):
    return _cabi.FsOrthOptions(*coefficients, eps, steps, products)


def matrices(*shapes, ld=None, src=FAKE, dst=FAKE * 2):
    rows = (_cabi.FsMatrix * len(shapes))()
    for row, (b, m, n) in zip(rows, shapes):
        row.src, row.dst, row.batch, row.rows, row.cols = src, dst, b, m, n
        row.src_ld = row.dst_ld = ld or n
        row.src_stride = row.dst_stride = m * (ld or n)
    return rows


def workspace(rows, opt):
    size = ctypes.c_int64(-1)
    rc = L.fsadam_orth_workspace(rows, len(rows), ctypes.byref(opt), ctypes.byref(size))
    return rc, size.value


def up(v, m):
    return (v + m - 1) // m * m


@pytest.mark.parametrize("products", [1, 2])
def test_workspace_holds_two_x_and_the_square_matrices_of_every_matrix(products):
    rc, got = workspace(matrices((3, 300, 170), (1, 135, 200)), options(products=products))
    assert rc == 0
    x = lambda s, l: 2 * 2 * up(s, 64) * up(l, 64) * 2  # two buffers of two planes of halves
    a = lambda s: (3 if products == 2 else 2) * products * up(s, 64) ** 2 * 2  # 22 bits: two planes, and steps in pairs need a third matrix
    body = 3 * (x(170, 300) + a(170)) + x(135, 200) + a(135)
    assert body < got < body + 4096  # and the tables


def test_workspace_of_a_long_list_stays_within_the_budget():
    one = workspace(matrices((1, 4096, 4096)), options())[1]
    rc, many = workspace(matrices(*[(1, 4096, 4096)] * 100), options())
    assert rc == 0 and one < many <= 4 << 30
    assert workspace(matrices((100, 4096, 4096)), options())[1] <= 4 << 30
    rc, big = workspace(matrices((1, 32768, 32768)), options())  # a matrix over the budget gets what it needs
    assert rc == 0 and big > 4 << 30


def test_empty_lists_and_matrices_need_nothing():
    assert workspace(matrices(), options()) == (0, 0)
    assert workspace(matrices((0, 4, 4), (1, 0, 4), (1, 4, 0)), options()) == (0, 0)
    opt = options()
    assert L.fsadam_orthogonalize(matrices((1, 0, 4)), 1, 0, ctypes.byref(opt), None, 0, None) == 0
    assert L.fsadam_orthogonalize(None, 0, 0, ctypes.byref(opt), None, 0, None) == 0
    assert L.fsadam_muon_step(None, 0, 0, 0, -1, ctypes.byref(opt), 0.1, 0.9, 1, 0.0, 1.0, None, None, 0, None) == 0


@pytest.mark.parametrize("bad", [
    dict(steps=0), dict(steps=33), dict(eps=0.0), dict(eps=-1.0), dict(eps=math.inf), dict(eps=math.nan), dict(products=0), dict(products=3),
    dict(coefficients=(math.nan, 0, 0)), dict(coefficients=(math.inf, 0, 0)),
    dict(coefficients=(30.0, 0.0, 0.0)),       # 30^5
    dict(coefficients=(1.0, 0.0, 5.0), steps=8),
])
def test_bad_options_are_refused(bad):
    rc, _ = workspace(matrices((1, 4, 4)), options(**bad))
    assert rc == -1 and L.fsadam_last_error()


@pytest.mark.parametrize("good", [
    dict(coefficients=(1.5, -0.5, 0.0)), dict(coefficients=(1.875, -1.25, 0.375)), dict(coefficients=(0.0, 0.0, 0.0)), dict(coefficients=(-3.4445, 4.7750, -2.0315)),
    dict(coefficients=(1.0, 0.0, 0.0), steps=32), dict(eps=1e-30), dict(coefficients=(2.0, -1.5, 0.5), steps=32),
])
def test_other_iterations_are_taken(good):
    assert workspace(matrices((1, 4, 4)), options(**good))[0] == 0


@pytest.mark.parametrize("rows, message", [
    (matrices((-1, 4, 4)), "negative"), (matrices((1, -4, 4)), "negative"), (matrices((1, 4, -4)), "negative"),
    (matrices((1, (1 << 20) + 1, 4)), "2^20"), (matrices((1, 1 << 20, 1 << 20)), "2^34"),
    (matrices((1, 4, 4), src=0), "NULL"), (matrices((1, 4, 4), dst=0), "NULL"), (matrices((1, 4, 4), ld=3), "overlap"),
])
def test_bad_matrices_are_refused(rows, message):
    rc, _ = workspace(rows, options())
    assert rc == -1 and message in L.fsadam_last_error().decode()


def test_bad_strides_alignment_and_workspaces_are_refused():
    opt = options()
    rows = matrices((2, 4, 4))
    rows[0].dst_stride = 15
    assert L.fsadam_orthogonalize(rows, 1, 0, ctypes.byref(opt), FAKE, 1 << 20, None) == -1
    rows = matrices((1, 4, 4), src=FAKE + 2)
    assert L.fsadam_orthogonalize(rows, 1, 0, ctypes.byref(opt), FAKE, 1 << 20, None) == -1 and b"aligned" in L.fsadam_last_error()
    rows = matrices((1, 4, 4), src=FAKE, dst=FAKE)
    rows[0].dst_ld = 8
    assert L.fsadam_orthogonalize(rows, 1, 0, ctypes.byref(opt), FAKE, 1 << 20, None) == -1 and b"same strides" in L.fsadam_last_error()
    rows = matrices((1, 200, 200))
    size = workspace(rows, opt)[1]
    assert L.fsadam_orthogonalize(rows, 1, 0, ctypes.byref(opt), None, size, None) == -1 and b"workspace" in L.fsadam_last_error()
    assert L.fsadam_orthogonalize(rows, 1, 0, ctypes.byref(opt), FAKE, size - 1, None) == -1 and b"workspace" in L.fsadam_last_error()
    assert L.fsadam_orthogonalize(rows, 1, 0, ctypes.byref(opt), FAKE + 16, size, None) == -1
    assert L.fsadam_orthogonalize(rows, 1, 3, ctypes.byref(opt), FAKE, size, None) == -1
    assert L.fsadam_orthogonalize(rows, 1, 0, None, FAKE, size, None) == -1
    assert L.fsadam_orth_workspace(rows, 1, ctypes.byref(opt), None) == -1
    assert L.fsadam_orth_workspace(None, 1, ctypes.byref(opt), ctypes.byref(ctypes.c_int64())) == -1


def muon_rows(**change):
    rows = (_cabi.FsMuonTensor * 1)()
    r = rows[0]
    r.p, r.g, r.m, r.p_copy, r.batch, r.rows, r.cols, r.ratio = FAKE, FAKE * 2, FAKE * 3, FAKE * 4, 1, 4, 4, 1.0
    for k, v in change.items():
        setattr(r, k, v)
    return rows


@pytest.mark.parametrize("call", [
    dict(types=(1, 0, -1)), dict(types=(0, 1, -1)), dict(types=(0, 1, 2)), dict(types=(0, 0, 0)), dict(types=(3, 3, -1)), dict(types=(1, 2, -1)),
    dict(lr=math.nan), dict(lr=math.inf), dict(weight_decay=math.inf), dict(momentum=1.0), dict(momentum=-0.1), dict(momentum=math.nan),
    dict(scale=0.0), dict(scale=math.inf), dict(scale=math.nan),
    dict(rows=muon_rows(p=0)), dict(rows=muon_rows(g=0)), dict(rows=muon_rows(m=0)), dict(rows=muon_rows(p_copy=0), types=(0, 1, 1)),
    dict(rows=muon_rows(m=FAKE + 2)), dict(rows=muon_rows(p=FAKE + 2)), dict(rows=muon_rows(ratio=math.nan)), dict(rows=muon_rows(rows=-1)),
    dict(rows=muon_rows(rows=200, cols=200), bytes=100),
])
def test_bad_steps_are_refused(call):
    opt = options()
    p, g, c = call.get("types", (0, 0, -1))
    rc = L.fsadam_muon_step(call.get("rows", muon_rows()), 1, p, g, c, ctypes.byref(opt), call.get("lr", 0.1), call.get("momentum", 0.9), 1,
                            call.get("weight_decay", 0.0), call.get("scale", 1.0), None, FAKE, call.get("bytes", 0), None)
    assert rc == -1 and L.fsadam_last_error()


def momentum_rows(**change):
    rows = (_cabi.FsMomentumTensor * 1)()
    r = rows[0]
    r.g, r.m, r.u, r.numel = FAKE, FAKE * 2, FAKE * 3, 10
    for k, v in change.items():
        setattr(r, k, v)
    return rows


@pytest.mark.parametrize("call", [
    dict(rows=momentum_rows(g=0)), dict(rows=momentum_rows(m=0)), dict(rows=momentum_rows(u=0)), dict(rows=momentum_rows(numel=-1)),
    dict(rows=momentum_rows(numel=1 << 43)), dict(rows=momentum_rows(g=FAKE + 2)), dict(types=(0, 3)), dict(types=(-1, 0)), dict(momentum=1.5),
    dict(scale=0.0), dict(bytes=100), dict(rows=momentum_rows(u=FAKE), types=(0, 1)),
])
def test_bad_momentum_passes_are_refused(call):
    g, u = call.get("types", (0, 0))
    rc = L.fsadam_momentum_pass(call.get("rows", momentum_rows()), 1, g, u, call.get("momentum", 0.9), 1, call.get("scale", 1.0), None, None, None, 0, FAKE,
                                call.get("bytes", 100), None)
    assert rc == -1 and L.fsadam_last_error()


def test_python_layer_refuses_what_is_not_on_a_gpu():
    with pytest.raises(RuntimeError, match="device"):
        orthogonalize([torch.zeros(4, 4)])
    with pytest.raises(RuntimeError, match="device"):
        momentum_pass([torch.zeros(4)], [torch.zeros(4)])
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        orthogonalize([torch.zeros(4, 4, dtype=torch.float64)])
    with pytest.raises(RuntimeError, match="same length"):
        momentum_pass([torch.zeros(4)], [])
    with pytest.raises(RuntimeError, match="at least one"):
        momentum_pass([], [])
    with pytest.raises(RuntimeError, match="as long"):
        orthogonalize([], out=[torch.zeros(1, 1)])
    assert orthogonalize([]) == []


def brute_layout(t):
    """What _layout promises, checked element by element against storage offsets."""
    got = matrix_ops._layout(t)
    if got is None:
        return None
    turned, ld, stride = got
    m = t.transpose(-2, -1) if turned else t
    offsets = torch.arange(t.untyped_storage().size() // t.element_size()).as_strided(m.shape, m.stride(), t.storage_offset())
    flat = offsets.reshape(-1, *m.shape[-2:])
    b, r, c = torch.meshgrid(*[torch.arange(n) for n in flat.shape], indexing="ij")
    assert torch.equal(flat, t.storage_offset() + b * stride + r * ld + c), (t.shape, t.stride(), got)
    assert ld >= m.shape[-1]
    return got


def test_layouts_describe_the_memory_they_are_read_from():
    base = torch.zeros(4, 6, 10)
    for t in (base, base.transpose(1, 2), base[:, :3], base[:, :, 2:7], base[:, 1:2], base[:, :, 4:5], base[1], base[1].t(), base[1:2], base[::2],
              base.view(2, 2, 6, 10), base.transpose(1, 2)[:, 3:4], base[:, 2:3, 3:4], base.view(2, 2, 6, 10)[:, :1], torch.zeros(1, 1), torch.zeros(1, 7), torch.zeros(7, 1),
              torch.zeros(7, 1).t(), torch.zeros(3, 1).expand(3, 1), torch.zeros(1, 4, 4).expand(5, 4, 4)):
        assert brute_layout(t) is not None, (t.shape, t.stride())
    for t in (base[:, :, ::2], base[:, ::2, ::2], torch.zeros(1, 4).expand(4, 4), base.view(2, 2, 6, 10).transpose(0, 1), base.view(2, 2, 6, 10)[:, :, :, ::3]):
        assert brute_layout(t) is None, (t.shape, t.stride())


def test_a_single_row_or_column_can_be_read_either_way():
    for t in (torch.zeros(5, 1), torch.zeros(1, 5), torch.zeros(5, 1).t(), torch.zeros(9, 9)[:, 2:3], torch.zeros(9, 9)[3:4]):
        turned = matrix_ops._layout(t)[0]
        other = matrix_ops._layout_as(t, not turned)
        if other is not None:
            m = t.transpose(-2, -1) if not turned else t
            assert other[0] is (not turned)
            assert m.shape[-1] == 1 or m.stride(-1) == 1
    assert matrix_ops._layout_as(torch.zeros(4, 5), True) is None


def test_optimizer_checks_its_arguments():
    w = lambda *s, dtype=torch.float32: [torch.nn.Parameter(torch.zeros(*s, dtype=dtype))]
    for bad in (dict(lr=-1.0), dict(lr=math.inf), dict(weight_decay=-1.0), dict(momentum=1.0), dict(momentum=-0.5), dict(eps=0.0), dict(ns_steps=0), dict(ns_steps=2.5),
                dict(ns_coefficients=(1.0, 2.0)), dict(ns_coefficients=(50.0, 0.0, 0.0)), dict(adjust_lr_fn="other"), dict(row_blocks=0), dict(row_blocks=3),
                dict(products="bf16"), dict(precision=Precision.PURE_FP16), dict(precision=Precision.MIXED_PRECISION)):
        with pytest.raises(ValueError):
            Muon(w(4, 4), **bad)
    with pytest.raises(ValueError, match="matrices"):
        Muon(w(4))
    with pytest.raises(ValueError, match="dtype"):
        Muon(w(4, 4) + w(4, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="FULL_PRECISION"):
        Muon(w(4, 4, dtype=torch.bfloat16), precision=Precision.FULL_PRECISION)
    opt = Muon(w(4, 4))
    assert opt.precision is Precision.FULL_PRECISION and opt.products == "split"
    opt = Muon(w(4, 4, dtype=torch.bfloat16))
    assert opt.precision is Precision.MIXED_PRECISION and opt.products == "split"
    assert opt.fp32_param_groups[0]["params"][0].dtype == torch.float32
    opt = Muon(w(4, 4, dtype=torch.bfloat16), precision=Precision.MEMORY_EFFICIENT_MIXED_PRECISION)
    assert opt.products == "half" and opt.fp32_param_groups == []
    with pytest.raises(ValueError):
        opt.add_param_group({"params": w(5, dtype=torch.bfloat16)})
    assert len(opt.param_groups) == 1


def test_optimizer_refuses_parameters_on_the_cpu_and_sparse_gradients():
    p = torch.nn.Parameter(torch.zeros(4, 4))
    opt = Muon([p])
    assert opt.step() is None  # no gradient: nothing to do
    p.grad = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="device tensors|one device"):
        opt.step()
    p.grad = torch.zeros(4, 4).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    assert torch.equal(p.detach(), torch.zeros(4, 4))


def test_state_of_16_bit_parameters_is_restored_bit_for_bit():
    p = torch.nn.Parameter(torch.randn(4, 4).to(torch.bfloat16))
    opt = Muon([p], lr=0.5)
    opt.state[p]["momentum_buffer"] = torch.randn(4, 4)
    opt.state[p]["master"] += 1e-5
    saved = opt.state_dict()
    other = Muon([torch.nn.Parameter(p.detach().clone())])
    other.load_state_dict(saved)
    q = other.param_groups[0]["params"][0]
    for key in ("momentum_buffer", "master"):
        assert torch.equal(other.state[q][key], opt.state[p][key]) and other.state[q][key].dtype == torch.float32
        assert other.state[q][key].data_ptr() != opt.state[p][key].data_ptr()
    assert other.fp32_param_groups[0]["params"][0] is other.state[q]["master"] and other.param_groups[0]["lr"] == 0.5


def test_oracle_agrees_with_singular_values():
    """The oracle's products against the polynomial on the singular values."""
    torch.manual_seed(0)
    u = torch.randn(2, 9, 5, dtype=torch.float64)
    a, b, c = M.COEFFICIENTS
    x, s, y = torch.linalg.svd(u, full_matrices=False)
    s = s / s.norm(dim=-1, keepdim=True)
    for _ in range(5):
        s = a * s + b * s**3 + c * s**5
    assert M.relative(M.orthogonal(u), x @ torch.diag_embed(s) @ y) < 1e-12


def test_workspace_of_matrices_that_fit_a_compute_unit():
    """They keep everything in LDS; only a long list's table needs memory."""
    assert workspace(matrices((1, 64, 256)), options()) == (0, 0)
    assert workspace(matrices((100, 128, 128), (7, 1, 64)), options()) == (0, 0)
    rc, got = workspace(matrices(*[(1, 96, 96)] * 25), options())
    assert rc == 0 and 0 < got < 8192
    assert workspace(matrices((1, 129, 129)), options())[1] > 0
    assert workspace(matrices((1, 64, 4096)), options())[1] > 0


def orth_row(src, dst, src_ld, dst_ld, shape=(3, 4), batch=1, src_stride=0, dst_stride=0):
    row = _cabi.FsMatrix()
    row.src, row.dst, row.batch = src, dst, batch
    row.rows, row.cols = shape
    row.src_ld, row.dst_ld, row.src_stride, row.dst_stride = src_ld, dst_ld, src_stride, dst_stride
    return row


@pytest.mark.parametrize("rows, apart", [
    ([orth_row(1000, 2000, 4, 4), orth_row(3000, 4000, 4, 4)], True),
    ([orth_row(1000, 1000, 4, 4), orth_row(2000, 2000, 4, 4)], True),                  # in place
    ([orth_row(1000, 2000, 4, 4), orth_row(1000, 3000, 4, 4)], True),                  # one matrix read twice
    ([orth_row(1000, 2000, 4, 4), orth_row(2000, 1000, 4, 4)], False),                 # exchanged
    ([orth_row(1000, 3000, 4, 4), orth_row(2000, 3000, 4, 4)], False),                 # the same result twice
    ([orth_row(1000, 1004, 4, 4)], False),                                             # shifted by an element
    ([orth_row(1000, 1000, 4, 8)], False),                                             # other strides
    ([orth_row(1000, 1000, 8, 8), orth_row(1016, 1016, 8, 8)], True),                  # halves of the columns
    ([orth_row(1000, 1000, 8, 8), orth_row(1012, 1012, 8, 8)], False),                 # they share a column
    ([orth_row(1000, 1000, 8, 8), orth_row(1020, 1020, 8, 8)], False),                 # the second runs into the next row
    ([orth_row(1000, 1000, 8, 8), orth_row(1016, 1016, 9, 9)], False),                 # not told apart
    ([orth_row(1000, 1000, 8, 8), orth_row(1018, 1018, 8, 8)], False),                 # not by whole elements
    ([orth_row(1000, 1000, 8, 8), orth_row(1048, 1048, 4, 4, (1, 4))], True),          # a single row in a gap
    ([orth_row(1000, 1000, 8, 8), orth_row(1044, 1044, 4, 4, (1, 4))], False),
    ([orth_row(1000, 1000, 8, 8, (3, 4), 2, 24, 24), orth_row(1016, 1016, 8, 8, (3, 4), 2, 24, 24)], True),
    ([orth_row(1000, 1000, 8, 8, (3, 4), 2, 28, 28), orth_row(1016, 1016, 8, 8, (3, 4), 2, 24, 24)], False),
    ([orth_row(1000, 1000, 4, 4, (1, 4), 5, 8, 8), orth_row(1016, 1016, 4, 4, (1, 4), 5, 8, 8)], True),
])
def test_results_that_share_memory_are_refused(rows, apart):
    if apart:
        matrix_ops._refuse_overlap(rows, 4)
    else:
        with pytest.raises(RuntimeError, match="shares memory"):
            matrix_ops._refuse_overlap(rows, 4)


def test_tensors_that_are_written_share_memory_with_nothing():
    base = torch.zeros(64)
    a, b, c = base[:16], base[16:32], base[8:24]
    matrix_ops.refuse_shared([a, b], [base[32:], base[40:]])
    matrix_ops.refuse_shared([a], [b, c[8:], torch.empty(0)])
    for written, read in (([a, a], []), ([a, c], []), ([a], [c]), ([c], [a]), ([b], [base]), ([base], [b])):
        with pytest.raises(RuntimeError, match="shares memory"):
            matrix_ops.refuse_shared(written, read)


def test_optimizer_looks_at_parameters_that_come_later():
    w = torch.nn.Parameter(torch.zeros(6, 4))
    opt = Muon([w], row_blocks=2)
    group = opt.param_groups[0]
    for bad in (torch.zeros(5), torch.zeros(5, 4)):
        p = torch.nn.Parameter(bad)
        with pytest.raises(ValueError):
            opt._check_shape(p, int(group["row_blocks"]))
    opt._check_group(group, 0)
    group["row_blocks"] = 4
    with pytest.raises(ValueError, match="cannot be split"):
        opt._check_group(group, 0)


def test_optimizer_is_copied_whole():
    w = torch.nn.Parameter(torch.randn(6, 4).half())
    opt = Muon([w], lr=0.5, products="half")
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        p = twin.param_groups[0]["params"][0]
        assert p is not w and torch.equal(p, w)
        assert (twin.precision, twin.products, twin.param_groups[0]["lr"]) == (Precision.MIXED_PRECISION, "half", 0.5)
        assert twin.fp32_param_groups[0]["params"][0] is twin.state[p]["master"] and torch.equal(twin.state[p]["master"], w.float())
        with pytest.raises(RuntimeError):
            p.grad = torch.zeros_like(p)
            twin.step()  # not on a GPU; gets as far as the check


# ---- master copies: what is saved is what is stepped ----------------------------------------------------------------

def mixed_optimizer(grad=True):
    p = torch.nn.Parameter(torch.randn(6, 4).to(torch.bfloat16))
    if grad:
        p.grad = torch.ones_like(p)
    return p, Muon([p])


def stepped(opt, p):
    """What the step of a parameter's group takes as parameter, momentum and copy."""
    parameters, _, momenta, copies = opt._gather(opt.param_groups[0])[p.device]
    return parameters[0], momenta[0], copies[0]


def test_a_state_assigned_to_a_parameter_is_the_one_that_is_stepped():
    """As OSS resumes: ``optimizer.state[p] = {...}``."""
    p, opt = mixed_optimizer()
    state = {"master": torch.full((6, 4), 7.0), "momentum_buffer": torch.full((6, 4), 3.0)}
    opt.state[p] = state
    assert all(a is b for a, b in zip(stepped(opt, p), (state["master"], state["momentum_buffer"], p)))
    assert opt.fp32_param_groups[0]["params"][0] is state["master"] is opt.state[p]["master"]
    assert opt.state_dict()["state"][0]["master"] is state["master"], "and the one that is saved"
    opt.state[p]["master"] = other = torch.full((6, 4), 8.0)
    assert stepped(opt, p)[0] is other and opt.fp32_param_groups[0]["params"][0] is other


@pytest.mark.parametrize("grad", [True, False])
def test_a_state_assigned_without_a_master_gets_one_from_the_parameter(grad):
    """As a checkpoint of another precision is restored; with or without a gradient by then."""
    p, opt = mixed_optimizer(grad)
    with torch.no_grad():
        p.fill_(5.0)
    opt.state[p] = {"momentum_buffer": torch.zeros(6, 4)}
    master = opt.fp32_param_groups[0]["params"][0]
    assert torch.equal(master, torch.full((6, 4), 5.0)) and master is opt.state[p]["master"] is opt.fp32_param_groups[0]["params"][0]
    if grad:
        assert stepped(opt, p)[0] is master


@pytest.mark.parametrize("bad", [torch.zeros(6, 4, dtype=torch.float16), torch.zeros(4, 6), torch.zeros(4, 6).t(), torch.zeros(6, 4, device="meta")], ids=["dtype", "shape", "strides", "device"])
def test_a_master_that_the_step_cannot_take_is_refused(bad):
    p, opt = mixed_optimizer()
    opt.state[p]["momentum_buffer"] = torch.zeros(6, 4)
    opt.state[p]["master"] = bad
    parameters, grads, momenta, copies = opt._gather(opt.param_groups[0])[p.device]
    assert parameters[0] is bad
    with pytest.raises(RuntimeError):
        opt.step()


def test_groups_of_masters_show_the_settings_in_use():
    p, opt = mixed_optimizer()
    opt.param_groups[0]["lr"] = 0.25
    assert opt.fp32_param_groups[0]["lr"] == 0.25


def test_a_master_that_nothing_steps_is_not_carried_on():
    """A checkpoint with masters restored without them, stepped, saved and restored with them again must not bring the old ones back."""
    p, opt = mixed_optimizer()
    saved = opt.state_dict()
    q = torch.nn.Parameter(p.detach().clone())
    other = Muon([q], precision=Precision.MEMORY_EFFICIENT_MIXED_PRECISION)
    other.load_state_dict(saved)
    assert "master" not in other.state_dict()["state"].get(0, {})
    other.state[q] = {"master": torch.zeros(6, 4), "momentum_buffer": torch.zeros(6, 4)}
    q.grad = torch.ones_like(q)
    stepped(other, q)
    assert "master" not in other.state_dict()["state"][0]


# ---- checkpoints ------------------------------------------------------------------------------------------------------

def test_a_checkpoint_of_torchs_optimizer_is_taken():
    """Its groups have no ``row_blocks``: what a checkpoint does not hold stays as this program has it."""
    p, q = torch.nn.Parameter(torch.randn(6, 4)), torch.nn.Parameter(torch.randn(5, 4))
    theirs = torch.optim.Muon([{"params": [p]}, {"params": [q], "lr": 0.5}], lr=0.25, momentum=0.75)
    p.grad, q.grad = torch.randn(6, 4), torch.randn(5, 4)
    theirs.step()
    saved = theirs.state_dict()
    assert "row_blocks" not in saved["param_groups"][0]
    ours = Muon([{"params": [torch.nn.Parameter(p.detach().clone())], "row_blocks": 3}, {"params": [torch.nn.Parameter(q.detach().clone())]}])
    ours.load_state_dict(saved)
    assert [(g["lr"], g["momentum"], g["row_blocks"]) for g in ours.param_groups] == [(0.25, 0.75, 3), (0.5, 0.75, 1)]
    for group, w in zip(ours.param_groups, (p, q)):
        assert torch.equal(ours.state[group["params"][0]]["momentum_buffer"], theirs.state[w]["momentum_buffer"])
        ours._check_group(group, 0)


@pytest.mark.parametrize("precision", [Precision.MIXED_PRECISION, Precision.MEMORY_EFFICIENT_MIXED_PRECISION], ids=["mixed", "memory_efficient"])
@pytest.mark.parametrize("change", [dict(lr=-1.0), dict(momentum=1.0), dict(eps=0.0), dict(adjust_lr_fn="other"), dict(row_blocks=4), dict(ns_steps=0),
                                    dict(ns_coefficients=(50.0, 0.0, 0.0)), dict(lr=None), "group", "parameter", "state"], ids=str)
def test_a_refused_checkpoint_changes_nothing(precision, change):
    def make():
        p, q = torch.nn.Parameter(torch.randn(6, 4).half()), torch.nn.Parameter(torch.randn(6, 4).half())
        opt = Muon([{"params": [p], "row_blocks": 2}, {"params": [q]}], lr=0.5, precision=precision)
        for w in (p, q):
            opt.state[w]["momentum_buffer"] = torch.randn(6, 4)
        return opt

    opt, other = make(), make()
    saved = copy.deepcopy(other.state_dict())
    saved["param_groups"][0]["lr"] = 0.125
    if change == "group":
        saved["param_groups"].pop()
    elif change == "parameter":
        saved["param_groups"][1]["params"].append(2)
    elif change == "state":
        saved["state"][1]["momentum_buffer"] = "missing"
    else:
        saved["param_groups"][1].update(change)
    groups, states = [dict(g) for g in opt.param_groups], {w: dict(st) for w, st in opt.state.items()}
    masters = [w for g in opt.fp32_param_groups for w in g["params"]]
    with pytest.raises((ValueError, TypeError, AttributeError)):
        opt.load_state_dict(saved)
    assert opt.param_groups == groups
    assert {w: dict(st) for w, st in opt.state.items()}.keys() == states.keys()
    assert all(opt.state[w][key] is value for w, st in states.items() for key, value in st.items())
    assert all(a is b for a, b in zip(masters, [w for g in opt.fp32_param_groups for w in g["params"]]))
    opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5


# ---- products of 11 bits ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("coefficients, steps, halves", [
    (M.COEFFICIENTS, 1, True), (M.COEFFICIENTS, 5, True), (M.COEFFICIENTS, 6, False), (M.COEFFICIENTS, 32, False), ((4.0848, -6.8946, 2.9270), 2, True),
    ((4.0848, -6.8946, 2.9270), 3, False), ((4.0848, -6.8946, 2.9270), 5, False), ((5.0, -20.0, 16.0), 2, False), ((1.5, -0.5, 0.0), 32, True), ((1.0, 0.0, 0.0), 5, True),
])
def test_11_bits_are_taken_where_their_error_stays_small(coefficients, steps, halves):
    """Otherwise the storage is that of 22 bits."""
    sizes = {p: workspace(matrices((1, 300, 500)), options(steps, coefficients, products=p))[1] for p in (1, 2)}
    assert (sizes[1] < sizes[2]) is halves and sizes[1] > 0


def test_bound_of_11_bit_products_holds_for_one_singular_value_with_the_roundings_made():
    x = torch.cat([torch.logspace(-3, 0, 300, dtype=torch.float64), torch.linspace(0.3, 1.0, 300, dtype=torch.float64)]).float().double()
    a, b, c = M.COEFFICIENTS

    def rounded(v):  # to 11 significant bits
        m, e = torch.frexp(v)
        return torch.ldexp(torch.round(m * 2048) / 2048, e)

    exact, held = x.clone(), x.clone()
    for _ in range(5):
        first = rounded(held)
        gram = rounded(first * first)
        held = a * held + rounded(b * gram + c * gram * gram) * first
        held = rounded(held) + rounded(held - rounded(held))
        exact = a * exact + b * exact**3 + c * exact**5
    error, bound = (held - exact).abs(), torch.tensor([M.half_bound(v, v) for v in x.tolist()])
    assert (error <= bound).all() and error.max() > 0.01, "and it is not far from what happens"


# ---- what a launch can hold -----------------------------------------------------------------------------------------------

def test_lists_longer_than_a_launch_are_refused_by_name():
    """A launch takes fewer than 2^32 threads; nothing of a call may be enqueued before that is known."""
    size = ctypes.c_int64()
    most = ((1 << 32) - 1) // 256 * 1024  # elements of the momentum pass: four to a thread
    for numel, rc in ((most, 0), (most + 1, -1), (1 << 40, -1)):
        rows = momentum_rows(numel=numel)
        assert L.fsadam_momentum_workspace(rows, 1, ctypes.byref(size)) == rc
        if rc:
            assert b"too many" in L.fsadam_last_error()
            assert L.fsadam_momentum_pass(rows, 1, 0, 0, 0.9, 1, 1.0, None, None, None, 0, FAKE, 1 << 40, None) == -1 and b"too many" in L.fsadam_last_error()
    halves = (_cabi.FsMomentumTensor * 2)()
    for row in halves:
        row.g, row.m, row.u, row.numel = FAKE, FAKE * 2, FAKE * 3, most // 2 + 1024
    assert L.fsadam_momentum_workspace(halves, 2, ctypes.byref(size)) == -1 and b"too many" in L.fsadam_last_error()
    many = (_cabi.FsMomentumTensor * (1 << 22))()  # one workgroup of 1024 threads to each norm
    assert L.fsadam_momentum_workspace(many, (1 << 22) - 1, ctypes.byref(size)) == 0
    assert L.fsadam_momentum_workspace(many, 1 << 22, ctypes.byref(size)) == -1 and b"too many" in L.fsadam_last_error()


def test_more_small_matrices_than_a_launch_holds_are_refused_by_name():
    opt = options()
    for shapes, rc in (([(1 << 20, 4, 4)] * 3 + [((1 << 20) - 1, 4, 4)], 0), ([(1 << 20, 4, 4)] * 4, -1)):
        rows = matrices(*shapes)
        assert workspace(rows, opt)[0] == rc
        if rc:
            assert b"too many" in L.fsadam_last_error()
            assert L.fsadam_orthogonalize(rows, len(rows), 0, ctypes.byref(opt), FAKE, 1 << 40, None) == -1 and b"too many" in L.fsadam_last_error()
    steps = (_cabi.FsMuonTensor * 4)()
    for row in steps:
        row.p, row.g, row.m, row.batch, row.rows, row.cols, row.ratio = FAKE, FAKE * 2, FAKE * 3, 1 << 20, 4, 4, 1.0
    size = ctypes.c_int64()
    assert L.fsadam_muon_workspace(steps, 4, ctypes.byref(opt), ctypes.byref(size)) == -1 and b"too many" in L.fsadam_last_error()
    assert L.fsadam_muon_step(steps, 4, 0, 0, -1, ctypes.byref(opt), 0.1, 0.9, 1, 0.0, 1.0, None, FAKE, 1 << 40, None) == -1 and b"too many" in L.fsadam_last_error()
    assert workspace(matrices(*[(1 << 20, 300, 300)] * 8), opt)[0] == 0  # these go through the workspace in chunks


# ---- numbers that do not fit their field ----------------------------------------------------------------------------------

@pytest.mark.parametrize("steps", [2**32 + 5, -(2**32) + 5, 2**31, 2**63, math.inf, math.nan, 5.5])
def test_steps_that_do_not_fit_are_refused(steps):
    """Not taken as what is left of them in 32 bits."""
    with pytest.raises(ValueError, match="steps"):
        matrix_ops.orth_options(steps, M.COEFFICIENTS, 1e-7, "split")
    with pytest.raises(ValueError, match="steps"):
        Muon([torch.nn.Parameter(torch.zeros(4, 4))], ns_steps=steps)


@pytest.mark.parametrize("change", [dict(lr=None), dict(momentum="much"), dict(ns_coefficients=5.0), dict(lr=-1.0), dict(row_blocks=math.inf)], ids=str)
def test_a_refused_group_is_not_added(change):
    opt = Muon([torch.nn.Parameter(torch.zeros(4, 4, dtype=torch.float16))])
    with pytest.raises((ValueError, TypeError, OverflowError)):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4, 4, dtype=torch.float16))], **change})
    assert len(opt.param_groups) == len(opt.fp32_param_groups) == len(opt.state) == 1
