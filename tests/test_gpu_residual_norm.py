"""Residual norm (kf_residual_norm_fwd / _bwd) against its formulas in float64.

Tolerance, max|a - b| / max(1, max|b|): 1e-5 for float32 tensors and 2e-2 for
bfloat16 ones, the framework's own.  A bfloat16 output is rounded once (2^-9); the
backward forms y again from x and the branch, without that rounding.  The float32 parameter gradients sum up to 4096
rows of float32 products: 4096 * 2^-24 = 2.4e-4 of the largest term at the very
worst, some 1e-6 of the result with errors of either sign.
"""

from __future__ import annotations

import pytest
import torch

import kanforge_b200 as kb

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 1e-5, torch.bfloat16: 2e-2}
NAMES = ("x", "branch", "weight", "bias", "branch_weight", "branch_bias", "gate")


def inputs(shape, kind, gate, branch_norm, dtype, branch_dtype=None, param_dtype=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    branch_dtype, param_dtype = branch_dtype or dtype, param_dtype or dtype
    width = shape[-1]
    t = {"x": (2 * r(*shape) + 0.5).to(dtype), "branch": r(*shape).to(branch_dtype),
         "weight": (1 + 0.2 * r(width)).to(param_dtype),
         "bias": (0.1 * r(width)).to(param_dtype) if kind == "layer" else None,
         "branch_weight": (1 + 0.2 * r(width)).to(param_dtype) if branch_norm else None,
         "branch_bias": (0.1 * r(width)).to(param_dtype) if branch_norm and kind == "layer" else None,
         "gate": None}
    if gate == "channel":
        t["gate"] = (0.5 * r(width)).to(param_dtype)
    elif gate == "token":
        t["gate"] = torch.sigmoid(r(*shape)).to(branch_dtype)
    elif gate == "sequence":  # broadcasts over the tokens of a sequence
        t["gate"] = torch.sigmoid(r(shape[0], 1, width)).to(branch_dtype)
    return t


def formula(t, kind, scale, eps):
    def norm(v):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        return v / (v.square().mean(-1, keepdim=True) + eps).sqrt()

    u = t["branch"]
    if t["branch_weight"] is not None:
        u = norm(u) * t["branch_weight"] + (0 if t["branch_bias"] is None else t["branch_bias"])
    y = scale * t["x"] + (u if t["gate"] is None else t["gate"] * u)
    return y, norm(y) * t["weight"] + (0 if t["bias"] is None else t["bias"])


def close(got, want, tol, what):
    assert got.shape == want.shape, what
    if got.numel() == 0:
        return
    err = (got.double() - want).abs().max().item() / max(1.0, want.abs().max().item())
    assert err <= tol, f"{what}: {err:.3e}"


def check(t, kind, scale, eps=1e-6, seed=1):
    leaves = {k: v.clone().requires_grad_() for k, v in t.items() if v is not None}
    y, h = kb.residual_norm(leaves["x"], leaves["branch"], leaves["weight"], leaves.get("bias"), kind=kind,
                            gate=leaves.get("gate"), branch_norm="branch_weight" in leaves,
                            branch_weight=leaves.get("branch_weight"), branch_bias=leaves.get("branch_bias"),
                            residual_scale=scale, eps=eps)
    assert y.dtype == t["x"].dtype and h.dtype == t["branch"].dtype
    g = torch.Generator(device="cuda").manual_seed(seed)
    dy = torch.randn(y.shape, generator=g, device="cuda").to(y.dtype)
    dh = torch.randn(h.shape, generator=g, device="cuda").to(h.dtype)
    grads = torch.autograd.grad([y, h], list(leaves.values()), [dy, dh])
    ref = {k: (v.double().requires_grad_() if v is not None else None) for k, v in t.items()}
    wy, wh = formula(ref, kind, scale, eps)
    want = torch.autograd.grad((wy * dy.double()).sum() + (wh * dh.double()).sum(), [ref[k] for k in leaves])
    close(y, wy.detach(), TOL[y.dtype], "y")
    close(h, wh.detach(), TOL[h.dtype], "h")
    low = torch.bfloat16 if torch.bfloat16 in {v.dtype for v in leaves.values()} else torch.float32
    for k, got, w in zip(leaves, grads, want):
        assert got.dtype == leaves[k].dtype
        close(got, w, TOL[low], k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("width", [1, 7, 8, 33, 768, 1000, 4096, 4097, 5000, 8192])
def test_matches_the_formulas_at_every_width(width, kind, dtype):
    check(inputs((37, width), kind, "channel", True, dtype), kind, 0.7, eps=1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("branch_norm", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "sequence"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gates_and_branch_norm(kind, gate, branch_norm, dtype):
    check(inputs((3, 41, 264), kind, gate, branch_norm, dtype), kind, 1.3)


@pytest.mark.parametrize("rows", [0, 1, 2, 4096])
def test_row_counts(rows):
    check(inputs((rows, 96), "layer", "channel", True, torch.float32), "layer", 1.0)


@pytest.mark.parametrize("param_dtype", [torch.float32, torch.bfloat16])
def test_float32_stream_with_bfloat16_branch(param_dtype):
    check(inputs((50, 512), "layer", "token", True, torch.float32, torch.bfloat16, param_dtype), "layer", 1.0)


def test_unaligned_and_strided_rows():
    t = inputs((20, 768), "layer", "channel", True, torch.bfloat16)
    wide = torch.zeros(20, 800, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:771] = t["x"]
    odd = torch.zeros(20 * 768 + 1, device="cuda", dtype=torch.bfloat16)
    odd[1:] = t["branch"].flatten()
    plain = kb.residual_norm(t["x"], t["branch"], t["weight"], t["bias"])
    views = kb.residual_norm(wide[:, 3:771], odd[1:].view(20, 768), t["weight"], t["bias"])
    for a, b in zip(plain, views):
        close(a, b.double(), 2e-2, "unaligned")


def test_large_mean_keeps_its_digits():
    # mean 1000, spread 1: squares about zero would lose 6 digits; about the mean they lose those of x itself
    x = torch.randn(8, 3000, device="cuda") + 1000.0
    _, h = kb.residual_norm(x, None, torch.ones(3000, device="cuda"), torch.zeros(3000, device="cuda"))
    d = x.double() - x.double().mean(-1, keepdim=True)
    want = d / (d.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    # x - mean is exact to the rounding of the mean (1000 * 2^-24 = 6e-5)
    assert (h.double() - want).abs().max() < 5e-4


def test_first_norm_and_missing_gradients():
    x = torch.randn(30, 200, device="cuda", requires_grad=True)
    w = torch.ones(200, device="cuda", requires_grad=True)
    y, h = kb.residual_norm(x, None, w, kind="rms")
    assert y is x
    want = torch.autograd.grad((x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w).square().sum(), [x, w])
    for a, b in zip(torch.autograd.grad(h.square().sum(), [x, w]), want):
        close(a, b.double(), 1e-5, "first norm")
    b = torch.randn(30, 200, device="cuda", requires_grad=True)
    y, h = kb.residual_norm(x, b, w, kind="rms", residual_scale=0.5)
    gx, gb = torch.autograd.grad(y.sum(), [x, b], retain_graph=True)  # nothing reaches h
    assert torch.equal(gx, torch.full_like(gx, 0.5)) and torch.equal(gb, torch.ones_like(gb))
    gx, gb = torch.autograd.grad(h.sum(), [x, b])  # nothing reaches y
    close(gx, 0.5 * gb.double(), 1e-6, "x and branch")


def test_gradient_matches_differences():
    t = inputs((4, 24), "layer", "token", True, torch.float32)
    args = {k: v.clone().requires_grad_() for k, v in t.items() if v is not None}

    def loss(a):
        y, h = kb.residual_norm(a["x"], a["branch"], a["weight"], a["bias"], gate=a["gate"], branch_norm=True,
                                branch_weight=a["branch_weight"], branch_bias=a["branch_bias"])
        return (y.double().sin().sum() + h.double().cos().sum())

    grads = torch.autograd.grad(loss(args), list(args.values()))
    for (name, v), g in zip(args.items(), grads):
        d = torch.randn_like(v)
        d /= d.norm()
        step = 2e-2  # central differences: step^2 against 2^-24 * |loss| / step
        with torch.no_grad():
            hi = loss({**args, name: v + step * d})
            lo = loss({**args, name: v - step * d})
        assert abs((hi - lo).item() / (2 * step) - (g.double() * d.double()).sum().item()) < 2e-2, name


def test_same_bits_every_run_and_on_another_stream():
    t = inputs((3000, 768), "layer", "channel", True, torch.bfloat16)

    def step():
        leaves = [t[k].clone().requires_grad_() for k in NAMES]
        x, b, w, s, bw, bs, g = leaves
        y, h = kb.residual_norm(x, b, w, s, gate=g, branch_norm=True, branch_weight=bw, branch_bias=bs)
        return [y, h, *torch.autograd.grad([y, h], leaves, [b.detach(), x.detach()])]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_a_bad_row_stays_in_its_row():
    t = inputs((9, 768), "layer", "channel", False, torch.float32)
    ref = kb.residual_norm(t["x"], t["branch"], t["weight"], t["bias"], gate=t["gate"])
    t["x"][4, 100] = float("nan")
    t["branch"][6, 3] = float("inf")
    got = kb.residual_norm(t["x"], t["branch"], t["weight"], t["bias"], gate=t["gate"])
    keep = [i for i in range(9) if i not in (4, 6)]
    for a, b in zip(got, ref):
        assert torch.equal(a[keep], b[keep])
    assert got[1][4].isnan().all() and got[1][6].isnan().any()


def test_module_trains():
    m = kb.ResidualNorm(64, "layer", branch_norm=True, gate_init=0.1, device="cuda")
    assert {n for n, _ in m.named_parameters()} == {"weight", "bias", "branch_weight", "branch_bias", "gate"}
    y, h = m(torch.randn(5, 64, device="cuda"), torch.randn(5, 64, device="cuda"))
    (y.sum() + h.square().sum()).backward()
    assert all(p.grad is not None for p in m.parameters())


def test_refusals():
    x = torch.randn(4, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    for bad, kind in [(dict(kind="batch"), ValueError), (dict(eps=-1.0), ValueError), (dict(branch_norm=True), ValueError),
                      (dict(branch_weight=w), ValueError)]:
        with pytest.raises(kind):
            kb.residual_norm(x, x, w, **bad)
    with pytest.raises(ValueError):
        kb.residual_norm(x, x[:2], w)
    with pytest.raises(ValueError):
        kb.residual_norm(x, None, w, gate=w)
    with pytest.raises(ValueError):
        kb.residual_norm(x, x, w[:8])
    with pytest.raises(TypeError):
        kb.residual_norm(x.bfloat16(), x, w)
    with pytest.raises(TypeError):
        kb.residual_norm(x.half(), x.half(), w.half())
    with pytest.raises(ValueError):
        kb.residual_norm(torch.randn(2, 8200, device="cuda"), None, torch.ones(8200, device="cuda"))
    with pytest.raises(RuntimeError):
        kb.residual_norm(x.cpu(), x.cpu(), w.cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(2371, 200), (1203, 512), (801, 768), (597, 1024), (483, 1280), (301, 2048), (397, 3000),
                                        (151, 4096), (103, 6144), (81, 8192)])
def test_many_rows(rows, width, dtype):
    """Enough rows for each group of warps to walk over several, by every number of warps to a row."""
    check(inputs((rows, width), "layer", "token", True, dtype), "layer", 0.9)
    check(inputs((rows, width), "rms", "channel", False, dtype), "rms", 1.0)


@pytest.mark.parametrize("width", [768, 4096])
def test_repeats_to_the_bit(width):
    t = inputs((3000, width), "layer", "channel", True, torch.bfloat16)
    g = torch.randn(3000, width, device="cuda").bfloat16()

    def run():
        leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
        y, h = kb.residual_norm(leaves["x"], leaves["branch"], leaves["weight"], leaves["bias"], gate=leaves["gate"],
                                branch_norm=True, branch_weight=leaves["branch_weight"], branch_bias=leaves["branch_bias"])
        return [y, h, *torch.autograd.grad([y, h], list(leaves.values()), [g, g])]

    for a, b in zip(run(), run()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [256 * chunks - 8 for chunks in range(1, 33)] + [3200, 6656])
def test_many_rows_at_every_division_of_a_row(width, dtype):
    """A row is 1 to 32 chunks of 256 elements, divided among lanes and warps; enough rows (2368 chunks) for groups
    that walk over several."""
    rows = -(-148 * 16 // -(-width // 256)) + 3
    check(inputs((rows, width), "layer", "channel", True, dtype), "layer", 0.9)


def test_saved_tensors_in_another_layout():
    t = inputs((40, 96), "layer", "token", True, torch.float32)
    grads = []
    for unpack in (lambda v: v, lambda v: v.transpose(0, -1).contiguous().transpose(0, -1)):
        leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, unpack):
            y, h = kb.residual_norm(leaves["x"], leaves["branch"], leaves["weight"], leaves["bias"], gate=leaves["gate"],
                                    branch_norm=True, branch_weight=leaves["branch_weight"], branch_bias=leaves["branch_bias"])
        grads.append(torch.autograd.grad([y, h], list(leaves.values()), [t["x"], t["branch"]]))
    for a, b in zip(*grads):
        assert torch.equal(a, b)
