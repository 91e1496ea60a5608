"""The mixing rule + LayerNorm on a GPU against its definition in 64 bits, forward and backward.

Bounds.  All arithmetic is fp32 on inputs that are read exactly; a row's sums are at most 16 additions in a thread and
then a tree.  s is off by E_s = 2^-21 (|G o| + |(1 - G) u|) (1 + |gate|) (the exponential's error grows with its argument),
mean and deviation by 2^-20 of the row's largest |s| (c), so xh by q = 2^-19 c rstd (1 + |xh|), and y by q |w| + 2^-23 |y| and one
rounding to its type, half a step.  A gradient is a product of such factors: with A the largest |a| of the row,
ds by 32 q rstd A (1 + |xh|)^2 taken with the row's largest |xh|, carried through the remaining factors, plus half a step.
Column sums add the rows' bounds and fp32 additions (a step per row and thread, at most rows + 64 steps of 2^-24).
"""

import threading

import pytest
import torch

from rnn_with_grm_b200 import cabi, cuda_ops
from rnn_with_grm_b200.fusion import fuse_layer_norm

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def make(rows, H, dtype, gate, scale, affine=True, param=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device=DEV, generator=g) * std + mean

    param = dtype if param is None else param
    return {"online": rand(rows, H).to(dtype), "update": rand(rows, H, std=0.7).to(dtype),
            "gate": rand(rows, H, std=2.0).to(dtype) if gate else None,
            "scale": rand(H, std=0.2, mean=1.0).to(param) if scale else None,
            "weight": rand(H, std=0.2, mean=1.0).to(param) if affine else None,
            "bias": rand(H, std=0.2).to(param) if affine else None}


def call(t, return_sum=False, eps=1e-5):
    return fuse_layer_norm(t["online"], t["update"], t["weight"], t["bias"], gate=t["gate"], scale=t["scale"], eps=eps,
                           return_sum=return_sum)


def reference(t, dy, dsum, eps=1e-5):
    """Outputs, gradients and the bounds on them, from the formulas in 64 bits."""
    w = {k: None if v is None else v.detach().double() for k, v in t.items()}
    o, b = w["online"], w["update"]
    H = o.shape[1]
    one = torch.ones(H, device=o.device, dtype=torch.float64)
    k = one if w["scale"] is None else w["scale"]
    u = b * k
    if w["gate"] is not None:
        G = torch.sigmoid(w["gate"])
        N, steep = torch.sigmoid(-w["gate"]), 1 + w["gate"].abs()
    else:
        G = N = torch.ones_like(o)
        steep = torch.ones_like(o)
    s = G * o + N * u
    s_tol = 2.0 ** -21 * ((G * o).abs() + (N * u).abs()) * steep
    mean = s.mean(1, keepdim=True)
    var = ((s - mean) ** 2).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (s - mean) * rstd
    top = (s.abs().amax(1, keepdim=True) + s_tol.amax(1, keepdim=True) * 2.0 ** 20)
    q = 2.0 ** -19 * top * rstd * (1 + xh.abs())
    lw = one if w["weight"] is None else w["weight"]
    lb = 0 * one if w["bias"] is None else w["bias"]
    y = xh * lw + lb
    half = HALF_STEP.get(t["online"].dtype, 0.0)
    out = {"y": y, "sum": s}
    tol = {"y": q * lw.abs() + 2.0 ** -22 * (y.abs() + lb.abs()) + half * 1.01 * y.abs(), "sum": s_tol + half * 1.01 * s.abs()}
    dy = torch.zeros_like(o) if dy is None else dy.double()
    a = dy * lw
    dx = rstd * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    big = a.abs().amax(1, keepdim=True)
    peak = 1 + xh.abs().amax(1, keepdim=True)
    e = 32 * q.amax(1, keepdim=True) * rstd * big * peak ** 2 + 2.0 ** -20 * rstd * big * peak ** 2
    e = e.expand_as(o)
    if dsum is not None:
        dx = dx + dsum.double()
        e = e + 2.0 ** -23 * dx.abs()
    du, du_tol = dx * (N if w["gate"] is not None else 1), e * N + 2.0 ** -20 * steep * dx.abs() * N
    out["online"], tol["online"] = dx * G, e * G + 2.0 ** -20 * steep * (dx * G).abs()
    out["update"], tol["update"] = du * k, du_tol * k.abs() + 2.0 ** -23 * (du * k).abs()
    if w["gate"] is not None:
        out["gate"] = dx * (o - u) * G * N
        tol["gate"] = (e * (o - u).abs() + 2.0 ** -19 * steep * dx.abs() * ((o - u).abs() + 2.0 ** -3 * (o.abs() + u.abs()))) * G * N
    for name in ("online", "update", "gate"):
        if name in out:
            tol[name] = tol[name] + half * 1.01 * out[name].abs()
    adds = (len(o) + 64) * 2.0 ** -24
    columns = {"weight": (dy * xh, dy.abs() * q), "bias": (dy, 0 * dy), "scale": (du * b, du_tol * b.abs())}
    for name, (terms, terms_tol) in columns.items():
        if w[name] is not None:
            out["p_" + name] = terms.sum(0)
            tol["p_" + name] = (terms_tol + adds * terms.abs()).sum(0) + HALF_STEP.get(t[name].dtype, 0.0) * 1.01 * terms.sum(0).abs()
    return out, tol


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    over = ((got.detach().double() - want).abs() - tol).max()
    assert torch.isfinite(got).all() and float(over) <= 1e-30, f"{what}: {float(over):.3e} over its bound"


def check(t, with_sum=False, use_dy=True, seed=1):
    dtype = t["online"].dtype
    g = torch.Generator(device=DEV).manual_seed(seed)
    dy = torch.randn(t["online"].shape, device=DEV, generator=g).to(dtype)
    dsum = torch.randn(t["online"].shape, device=DEV, generator=g).to(dtype) if with_sum else None
    names = [k for k in ("online", "update", "gate", "scale", "weight", "bias") if t[k] is not None]
    if not use_dy:
        names = [k for k in names if k not in ("weight", "bias")]
    for k in names:
        t[k].requires_grad_(True)
    got = call(t, with_sum)
    want, tol = reference(t, dy if use_dy else None, dsum)
    y, total = got if with_sum else (got, None)
    within(y, want["y"], tol["y"], "y")
    if with_sum:
        within(total, want["sum"], tol["sum"], "sum")
    outs, ups = ([y] if use_dy else []) + ([total] if with_sum else []), ([dy] if use_dy else []) + ([dsum] if with_sum else [])
    for k, grad in zip(names, torch.autograd.grad(outs, [t[k] for k in names], ups)):
        assert grad.dtype == t[k].dtype
        key = "p_" + k if k in ("scale", "weight", "bias") else k
        within(grad, want[key], tol[key], "gradient of " + k)


SIZES = [(1, 1), (3, 2), (5, 17), (8, 512), (33, 64), (65, 513), (100, 512), (7, 1000), (19, 2048), (6, 2056), (5, 8191), (3, 8192)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("rule", ["residual", "residual scaled", "gate", "gate scaled"])
@pytest.mark.parametrize("types", ["bf16", "bf16 fp32", "fp32"])
def test_outputs_and_gradients_match_the_definition(size, rule, types):
    rows, H = size
    dtype = torch.float32 if types == "fp32" else torch.bfloat16
    param = torch.bfloat16 if types == "bf16" else torch.float32
    t = make(rows, H, dtype, "gate" in rule, "scaled" in rule, param=param, seed=rows + H)
    check(t, with_sum=rows % 2 == 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H", [48, 515, 3000])
def test_many_rows_share_their_column_sums(dtype, H):
    check(make(5003, H, dtype, True, True, seed=H), with_sum=True)


def test_without_affine_and_with_the_sum_alone():
    check(make(40, 96, torch.float32, False, False, affine=False))
    check(make(40, 96, torch.bfloat16, True, True, affine=False), with_sum=True)
    check(make(40, 96, torch.float32, True, True), with_sum=True, use_dy=False)


def test_gradient_agrees_with_differences():
    t = make(12, 40, torch.float32, True, True, seed=2)
    c = torch.randn(12, 40, device=DEV)
    for k in t:
        v = torch.randn_like(t[k])
        t[k].requires_grad_(True)
        slope = float((torch.autograd.grad((call(t) * c).sum(), t[k])[0].double() * v).sum())
        t[k].requires_grad_(False)

        def along(h, wide=False):
            moved = dict(t, **{k: t[k].double() + h * v.double()})
            if not wide:
                moved[k] = moved[k].float()
                return float((call(moved).double() * c.double()).sum())
            return float((reference(moved, None, None)[0]["y"] * c.double()).sum())

        h = 2.0 ** -7
        estimate = (along(h) - along(-h)) / (2 * h)
        # the estimate's own error: Richardson's, from the definition in 64 bits, and the outputs' rounding
        e1, e2 = ((along(x, True) - along(-x, True)) / (2 * x) for x in (h, h / 2))
        bound = 2 * abs(e1 - e2) + 2.0 ** -18 * float((c.abs() * 8).sum()) / h / 40 + 1e-4 * abs(slope)
        assert abs(estimate - slope) <= bound, k


def test_agrees_with_the_inference_kernel():
    # the plain residual rule is what grmx_add_layer_norm computes; both round one fp32 result to bf16
    t = make(300, 512, torch.bfloat16, False, False, param=torch.float32, seed=3)
    want = torch.ops.grmx.add_layer_norm(t["online"], t["update"], t["weight"], t["bias"], 1e-5)
    step = 2.0 ** -7 * want.float().abs() + 2.0 ** -20
    assert ((call(t).float() - want.float()).abs() <= step).all()


def test_gates_at_their_ends_and_constant_rows():
    t = make(4, 64, torch.float32, True, False, seed=4)
    t["gate"][0], t["gate"][1] = float("inf"), float("-inf")
    y, total = call(t, return_sum=True)
    assert torch.equal(total[0], t["online"][0]) and torch.equal(total[1], t["update"][1])
    t["gate"].requires_grad_(True)
    (dg,) = torch.autograd.grad(call(t).sum() + call(t, return_sum=True)[1].sum(), t["gate"])
    assert not dg[:2].any() and torch.isfinite(dg).all()
    flat = {**make(2, 64, torch.float32, False, False), "online": torch.full((2, 64), 3.0, device=DEV), "update": torch.zeros(2, 64, device=DEV)}
    assert torch.equal(call(flat), flat["bias"].expand(2, 64))       # no deviation: the bias alone
    bad = make(3, 64, torch.float32, False, False)
    clean = call(bad)
    bad["online"][1, 5] = float("nan")
    assert torch.equal(call(bad)[[0, 2]], clean[[0, 2]]) and torch.isnan(call(bad)[1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_strides_alignment_and_leading_dimensions(dtype):
    t = make(24, 96, dtype, True, True, seed=5)
    want = call(t)
    moved = {}
    for k, v in t.items():
        moved[k] = torch.empty(v.numel() + 1, device=DEV, dtype=dtype)[1:].view(v.shape).copy_(v)
    # value by value instead of 16-byte pieces: a thread adds other columns, so sums differ in their last bits
    assert ((call(moved).float() - want.float()).abs() <= 2 * HALF_STEP[dtype] * want.float().abs() + 2.0 ** -18).all()
    shaped = {k: v.view(2, 3, 4, 96) if v.dim() == 2 else v for k, v in t.items()}
    assert torch.equal(call(shaped).view(24, 96), want)
    across = {k: v.T.contiguous().T if v.dim() == 2 else v for k, v in t.items()}
    assert torch.equal(call(across), want)


def test_no_rows():
    t = make(0, 64, torch.bfloat16, True, True)
    for v in t.values():
        v.requires_grad_(True)
    y = call(t)
    assert y.shape == (0, 64)
    for k, grad in zip(t, torch.autograd.grad(y.sum(), list(t.values()))):
        assert grad.shape == t[k].shape and not grad.any()


def test_only_the_gradients_that_are_asked_for():
    t = make(50, 96, torch.bfloat16, True, True, seed=6)
    dy = torch.randn(50, 96, device=DEV).bfloat16()
    for v in t.values():
        v.requires_grad_(True)
    every = dict(zip(t, torch.autograd.grad(call(t), list(t.values()), dy)))
    for k in t:
        for j, v in t.items():
            v.requires_grad_(j == k)
        assert torch.equal(torch.autograd.grad(call(t), t[k], dy)[0], every[k])


def test_same_bits_on_two_streams_and_in_a_captured_step():
    t = make(700, 512, torch.bfloat16, True, True, seed=7)
    dy = torch.randn(700, 512, device=DEV).bfloat16()
    for v in t.values():
        v.requires_grad_(True)

    def step():
        y = call(t)
        return (y.detach(), *torch.autograd.grad(y, list(t.values()), dy))

    first = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for r in results for p, q in zip(first, r))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    new = make(700, 512, torch.bfloat16, True, True, seed=8)
    with torch.no_grad():
        for k in t:
            t[k].copy_(new[k])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, step()))
    cuda_ops.check_device_errors()


def test_rows_behind_the_last_stay_as_they_are():
    lib = cabi.load()
    t = make(5, 100, torch.float32, False, False, seed=9)
    out = torch.full((8, 100), 7.0, device=DEV)
    cabi.check(lib.grmx_fuse_norm_fwd(cabi.ptr(t["online"]), cabi.ptr(t["update"]), None, None, cabi.ptr(t["weight"]),
                                      cabi.ptr(t["bias"]), 1e-5, cabi.ptr(out), None, None, 5, 100, cabi.F32, cabi.F32,
                                      cabi.current_stream()))
    torch.cuda.synchronize()
    assert torch.equal(out[:5], call(t)) and (out[5:] == 7.0).all()


# rows that are not a multiple of 16 bytes keep their parameters in shared memory: widths where these and the rows' own
# few hundred bytes meet 48 KiB, forward (three vectors) and backward (two)
@pytest.mark.parametrize("H", [3630, 3631, 3635, 3637, 3639, 3641, 5401, 5405, 5433, 5459, 5461, 5463])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_parameters_of_about_48_kib(dtype, H):
    check(make(5, H, dtype, True, True, seed=H), with_sum=True)


def test_threads_of_different_widths():
    inputs = [make(4, H, torch.bfloat16, True, True, seed=H) for H in (4105, 5001, 6007, 8001)]      # 54 to 106 KiB
    wants = [call(t) for t in inputs]
    failures = []

    def work(own):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(3000):
                    out = call(inputs[own[i % 2]])
                assert torch.equal(out, wants[own[1]])
        except Exception as e:  # noqa: BLE001 -- reported by the test's own thread
            failures.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(own,)) for own in ((0, 3), (1, 2), (2, 0), (3, 1))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H", [96, 1000, 8184, 8192])
def test_parameters_off_16_byte_boundaries(dtype, H):
    # rows that could move whole, beside parameters that cannot
    t = make(9, H, dtype, True, True, seed=H)
    for k in ("scale", "weight", "bias"):
        t[k] = torch.empty(H + 1, device=DEV, dtype=dtype)[1:].copy_(t[k])
    check(t, with_sum=True)


def test_offsets_beyond_32_bits():
    rows, H = 4_250_000, 512
    assert rows * H > 1 << 31
    t = make(rows, H, torch.bfloat16, False, False, seed=10)
    dy = torch.randn(300, H, device=DEV).bfloat16()
    ends = [slice(0, 300), slice(rows - 300, rows)]
    up = torch.zeros(rows, H, device=DEV, dtype=torch.bfloat16)
    for s in ends:
        up[s] = dy
    for k in ("online", "weight"):
        t[k].requires_grad_(True)
    y = call(t)
    d_online, d_weight = torch.autograd.grad(y, [t["online"], t["weight"]], up)
    total = torch.zeros(H, device=DEV, dtype=torch.float64)
    for s in ends:
        part = {k: None if v is None else v.detach()[s] if v.dim() == 2 else v.detach() for k, v in t.items()}
        want, tol = reference(part, dy, None)
        within(y[s], want["y"], tol["y"], "y")
        within(d_online[s], want["online"], tol["online"], "gradient of online")
        total += want["p_weight"]
    assert ((d_weight.double() - total).abs() <= 2.0 ** -7 * total.abs() + 1e-3).all()
    assert not d_online[300:-300].any()


def test_wide_rows_off_16_byte_boundaries_in_a_captured_step():
    t = make(40, 8001, torch.bfloat16, True, True, seed=11)
    dy = torch.randn(40, 8001, device=DEV).bfloat16()
    for v in t.values():
        v.requires_grad_(True)

    def step():
        y = call(t)
        return (y.detach(), *torch.autograd.grad(y, list(t.values()), dy))

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for v in out:
        v.zero_()
    call(make(4, 4105, torch.bfloat16, True, True))           # a narrower call in between
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_equal_gradients_are_two_tensors_of_their_leaves():
    # without gate and scale one row gradient is written for both
    t = make(30, 96, torch.bfloat16, False, False, seed=12)
    for k in ("online", "update"):
        t[k].requires_grad_(True)
    call(t).float().square().sum().backward()
    want = t["update"].grad.clone()
    assert torch.equal(t["online"].grad, want) and want.any()
    t["online"].grad.zero_()
    assert torch.equal(t["update"].grad, want)
