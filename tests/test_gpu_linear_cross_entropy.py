"""The vocabulary loss on a GPU against its definition in 64 bits.

Bounds.  A score is a sum of D products: bf16 products are exact in fp32 and every addition rounds by at most one
fp32 step (2^-23, also if it truncates), so |error of y_ij| <= e_ij = (D + 16) 2^-23 (sum_k |x_ik W_jk| + |b_j|); the six
plane products of full precision lose at most 3 x 2^-24 of each product on top, which the 16 covers at D >= 1 with
the joins and the base-2 scaling.  With e_i = max_j e_ij the loss is off by at most 2 e_i plus a few steps of the
logarithm; a probability by a factor of exp(2 e_i + 2^-20) (the exponential's own error is below 2^-21).  d = p - [target] is rounded
once to bf16 (2^-8 of itself; in full precision 2^-24, three planes) before it is multiplied; with a factor per token the
tokens that dW multiplies it with are rounded once more, x g to the same type; the products accumulate as
above -- over at most 128 + 8 additions between two roundings in full precision, over the whole contraction in
bf16 -- and the result is rounded once to its own type.
"""

import threading

import pytest
import torch

from rnn_with_grm_b200 import cabi, cuda_ops
from rnn_with_grm_b200.fusion import fuse_layer_norm
from rnn_with_grm_b200.loss import linear_cross_entropy
from rnn_with_grm_b200.segment_memory import StackedSegmentMemoryRunner, language_model_parameter_shapes

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def make(N, D, V, dtype, bias=None, ignored=0.0, seed=0, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, D, device=DEV, generator=g).to(dtype)
    w = (torch.randn(V, D, device=DEV, generator=g) * (std / D ** 0.5)).to(dtype)
    b = None if bias is None else torch.randn(V, device=DEV, generator=g).to(bias)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    if ignored:
        t = torch.where(torch.rand(N, device=DEV, generator=g) < ignored, torch.full_like(t, -100), t)
    return x, w, b, t


def reference(x, w, b, t, upstream, ignore_index=-100):
    """Loss per token, its gradients for the upstream gradient per token, and the bounds on all of them."""
    dtype = x.dtype
    X, W = x.detach().double(), w.detach().double()
    B = torch.zeros(len(W), device=X.device, dtype=torch.float64) if b is None else b.detach().double()
    D = X.shape[1]
    y = X @ W.T + B
    valid = t != ignore_index
    at = t.clamp(0, len(W) - 1)[:, None]
    lse = torch.logsumexp(y, 1)
    loss = torch.where(valid, lse - y.gather(1, at)[:, 0], torch.zeros_like(lse))
    size = X.abs() @ W.abs().T + B.abs().nan_to_num(posinf=0.0)
    e = (D + 16) * 2.0 ** -23 * size.amax(1)
    loss_tol = torch.where(valid, 2 * e + 2.0 ** -20 * (1 + loss.abs()), torch.zeros_like(e))
    p = torch.exp(y - lse[:, None])
    unit = p.clone()
    unit.scatter_add_(1, at, torch.full_like(lse, -1.0)[:, None])
    g = torch.where(valid, upstream.double(), torch.zeros_like(lse))
    d = unit * g[:, None]
    d_tol = g.abs()[:, None] * (p * (2 * e + 2.0 ** -20)[:, None] * 1.01 + HALF_STEP[dtype] * unit.abs())
    grads, tols = {}, {}
    for name, a, a_tol, other, length in (("x", d, d_tol, W, len(W)), ("w", d.T, d_tol.T, X, len(X))):
        grads[name] = a @ other
        steps = 136 + length * 6 / (64 * 32) if dtype == torch.float32 else length + 16
        weighted = HALF_STEP[dtype] if name == "w" and not torch.equal(upstream, upstream[:1].expand_as(upstream)) else 0.0
        tols[name] = (a_tol + (steps * 2.0 ** -23 + weighted) * a.abs()) @ other.abs() + 2 * HALF_STEP[dtype] * grads[name].abs()
    if b is not None:
        grads["b"] = d.sum(0)
        # sums of the same rounded d, in fp32 additions, 32 rows and then the blocks
        tols["b"] = (d_tol + (40 + len(X) / 32) * 2.0 ** -24 * d.abs()).sum(0) + 2 * HALF_STEP[b.dtype] * grads["b"].abs()
    return loss, loss_tol, grads, tols


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    over = ((got.detach().double() - want).abs() - tol).max()
    assert torch.isfinite(got).all() and float(over) <= 1e-30, f"{what}: {float(over):.3e} over its bound"


SHAPES = [(1, 1, 1), (1, 512, 1000), (2, 64, 256), (7, 33, 257), (127, 65, 255), (129, 8, 300), (256, 128, 512), (300, 72, 513),
          (513, 520, 777), (40, 1030, 130), (3, 100, 33), (8, 520, 3000), (9, 520, 3000), (4, 6000, 70), (260, 257, 300), (260, 384, 300), (260, 385, 300)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_loss_and_gradients_match_the_definition(shape, dtype, reduction):
    N, D, V = shape
    bias = {"none": None, "sum": dtype, "mean": torch.float32}[reduction]
    x, w, b, t = make(N, D, V, dtype, bias, ignored=0.2 if reduction != "sum" and N > 1 else 0.0, seed=N + D + V)
    if N > 1:
        t[0] = V - 1                                     # a token that counts, in the last column tile
    leaves = [v.requires_grad_(True) for v in (x, w, b) if v is not None]
    loss = linear_cross_entropy(x, w, t, b, reduction=reduction)
    count = int((t != -100).sum())
    if reduction == "none":
        up = torch.rand(N, device=DEV) + 0.5
        grads = torch.autograd.grad(loss, leaves, up)
    else:
        grads = torch.autograd.grad(loss * 1.5, leaves)
        up = torch.full((N,), 1.5 / (count if reduction == "mean" else 1), device=DEV)
    want, tol, want_grads, grad_tols = reference(x, w, b, t, up)
    if reduction != "none":
        scale = 1 / count if reduction == "mean" else 1
        want, tol = want.sum() * scale, tol.sum() * scale + 2.0 ** -23 * want.sum().abs() * scale
    assert loss.dtype == torch.float32
    within(loss, want, tol, "loss")
    for name, grad, leaf in zip("xwb", grads, leaves):
        assert grad.dtype == leaf.dtype
        # (1 / count and its product with the upstream gradient are rounded in fp32)
        within(grad, want_grads[name], grad_tols[name] + 2.0 ** -22 * want_grads[name].abs(), "gradient of " + name)
    cuda_ops.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(64, 40, 20000), (9000, 24, 300), (1500, 300, 5000)], ids=["many words", "many tokens", "both"])
def test_long_contractions_are_cut_and_joined(dtype, shape):
    x, w, b, t = make(*shape, dtype, torch.float32, ignored=0.1, seed=3)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    up = torch.rand(shape[0], device=DEV) + 0.5
    loss = linear_cross_entropy(x, w, t, b, reduction="none")
    grads = torch.autograd.grad(loss, leaves, up)
    want, tol, want_grads, grad_tols = reference(x, w, b, t, up)
    within(loss, want, tol, "loss")
    for name, grad in zip("xwb", grads):
        within(grad, want_grads[name], grad_tols[name], "gradient of " + name)


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (30011, 16, 18300)), (torch.float32, (16001, 16, 11500))], ids=["bf16", "fp32"])
def test_a_vocabulary_in_several_pieces(dtype, shape):
    N, D, V = shape
    planes = 1 if dtype == torch.bfloat16 else 3
    assert 2 * planes * N * V > 1 << 30                   # more than one piece
    x, w, b, t = make(N, D, V, dtype, dtype, ignored=0.1, seed=4)
    t[0], t[1] = 0, V - 1
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b, reduction="sum")
    grads = torch.autograd.grad(loss, leaves)
    rows = torch.arange(0, N, 31, device=DEV)             # every 31st token's own gradient
    want, _, want_grads, grad_tols = reference(x[rows], w, b, t[rows], torch.ones(len(rows), device=DEV))
    within(grads[0][rows], want_grads["x"], grad_tols["x"], "gradient of x")
    # the words' gradients over all tokens, a few hundred words at a time from every piece
    X, W, B = x.detach().double(), w.detach().double(), b.detach().double()
    lse = torch.cat([torch.logsumexp(torch.addmm(B, X[i:i + 2000], W.T), 1) for i in range(0, N, 2000)])
    valid = (t != -100).double()
    e = (D + 16) * 2.0 ** -23 * (X.abs().sum(1) * W.abs().max() + B.abs().max())
    for v0 in (0, V // 2 - 60, V - 120):
        words = torch.arange(v0, v0 + 120, device=DEV)
        p = torch.exp(X @ W[words].T + B[words] - lse[:, None])
        d = (p - (t[:, None] == words).double()) * valid[:, None]
        d_tol = p * (2 * e + 2.0 ** -20)[:, None] * 1.01 + HALF_STEP[dtype] * d.abs()
        steps = 136 + N * 6 / 2048 if dtype == torch.float32 else N + 16
        tol = (d_tol + steps * 2.0 ** -23 * d.abs()).T @ X.abs() + 2 * HALF_STEP[dtype] * (d.T @ X).abs()
        within(grads[1][words], d.T @ X, tol, f"gradient of words from {v0}")
        fine = (d_tol + (40 + N / 32) * 2.0 ** -24 * d.abs()).sum(0)
        within(grads[2][words], d.sum(0), fine + 2 * HALF_STEP[dtype] * d.sum(0).abs(), f"bias gradient of words from {v0}")


def test_gradient_agrees_with_differences():
    # |L(x + h v) - L(x - h v)| / 2h: the third derivative of a log-sum-exp along v is at most (range of v.W)^3, and the
    # losses are off by their own bound
    x, w, b, t = make(48, 40, 700, torch.float32, torch.float32, seed=5)
    _, tol, _, _ = reference(x, w, b, t, torch.ones(48, device=DEV))
    h = 2.0 ** -6
    for i, leaf in enumerate((x, w, b)):
        leaves = [x, w, b]
        v = torch.randn_like(leaf)
        v /= v.norm(dim=-1, keepdim=True)
        leaf.requires_grad_(True)
        loss = linear_cross_entropy(x, w, t, b, reduction="none")
        slope = float((torch.autograd.grad(loss.sum(), leaf)[0].double() * v).sum())
        leaf.requires_grad_(False)
        ends = []
        for sign in (1, -1):
            moved = list(leaves)
            moved[i] = leaf + sign * h * v
            ends.append(float(linear_cross_entropy(*moved[:2], t, moved[2], reduction="none").double().sum()))
        change = v @ w.T if i == 0 else x @ v.T if i == 1 else v.expand(48, -1)
        third = float(((change.amax(1) - change.amin(1)).double() ** 3).sum())
        bound = third * h * h / 6 + 2 * float(tol.sum()) / (2 * h) + 1e-4 * abs(slope)
        assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_masked_words_and_ignored_tokens(dtype):
    x, w, _, t = make(70, 64, 700, dtype, seed=6)
    b = torch.zeros(700, device=DEV)
    b[256:520] = float("-inf")                            # a whole column tile and more without a word
    b[3] = float("-inf")
    t = torch.where((t >= 256) & (t < 520) | (t == 3), torch.full_like(t, 100), t)
    t[5] = -7
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b, ignore_index=-7, reduction="none")
    grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    open_words = torch.isfinite(b)
    renamed = torch.cumsum(open_words, 0) - 1
    t_open = torch.where(t == -7, t, renamed[t.clamp(min=0)])
    want, tol, want_grads, grad_tols = reference(x, w[open_words], b[open_words], t_open, torch.ones(70, device=DEV), ignore_index=-7)
    within(loss, want, tol, "loss")
    within(grads[0], want_grads["x"], grad_tols["x"], "gradient of x")
    within(grads[1][open_words], want_grads["w"], grad_tols["w"], "gradient of w")
    assert float(loss.detach()[5]) == 0.0 and not grads[0][5].any()
    assert not grads[1][~open_words].any() and not grads[2][~open_words].any()


def test_no_token_counts():
    x, w, b, t = make(9, 64, 300, torch.bfloat16, torch.bfloat16, seed=7)
    t[:] = -100
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b)
    assert torch.isnan(loss)
    for grad in torch.autograd.grad(loss, leaves):
        assert not grad.any()
    assert float(linear_cross_entropy(x, w, t, b, reduction="sum").detach()) == 0.0
    assert not linear_cross_entropy(x, w, t, b, reduction="none").detach().any()


def test_no_tokens_at_all():
    x, w, b, t = make(0, 64, 300, torch.bfloat16, torch.bfloat16)
    assert linear_cross_entropy(x, w, t, b, reduction="none").shape == (0,)
    assert float(linear_cross_entropy(x, w, t, b, reduction="sum")) == 0.0 and torch.isnan(linear_cross_entropy(x, w, t, b))
    w.requires_grad_(True)
    (grad,) = torch.autograd.grad(linear_cross_entropy(x, w, t, b, reduction="sum"), w)
    assert not grad.any()


def test_values_that_are_not_finite_stay_in_their_rows():
    x, w, _, t = make(6, 64, 300, torch.bfloat16, seed=8)
    clean = linear_cross_entropy(x, w, t, reduction="none")
    x[1, 3] = float("nan")
    x[4, 7] = float("inf")
    loss = linear_cross_entropy(x, w, t, reduction="none")
    assert torch.isnan(loss[[1, 4]]).all() and torch.equal(loss[[0, 2, 3, 5]], clean[[0, 2, 3, 5]])
    closed = torch.full((300,), float("-inf"), device=DEV)
    assert torch.isnan(linear_cross_entropy(x, w, t, closed, reduction="none")).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_what_ignored_tokens_hold_goes_nowhere(dtype, reduction):
    x, w, b, t = make(300, 72, 513, dtype, dtype, ignored=0.3, seed=18)
    up = torch.rand(300, device=DEV) if reduction == "none" else None

    def step(x, up):
        x = x.clone().requires_grad_(True)
        leaves = [x, w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction=reduction)
        return (loss.detach(), *torch.autograd.grad(loss, leaves, up))

    clean = step(x, up)
    bad, skip = x.clone(), (t == -100).nonzero()[:, 0]
    bad[skip[0]] = float("nan")
    bad[skip[1], 3] = float("inf")
    if up is not None:
        up = up.clone()
        up[skip[2]], up[skip[3]] = float("inf"), float("nan")
    for p, q in zip(clean, step(bad, up)):
        assert torch.equal(p, q)


def test_large_scores_and_a_certain_target():
    # scores of +-4000: the sum of exponentials must not overflow, and a target that is the maximum by far has
    # a loss of exactly log(1) = 0
    w = torch.eye(64, device=DEV).bfloat16()
    x = torch.zeros(64, 64, device=DEV)
    x.fill_diagonal_(4000.0)
    x = x.bfloat16()
    t = torch.arange(64, device=DEV)
    assert not linear_cross_entropy(x, w, t, reduction="none").any()
    other = linear_cross_entropy(x, w, (t + 1) % 64, reduction="none")
    assert torch.equal(other, torch.full_like(other, float(x[0, 0])))


def test_target_outside_the_vocabulary_is_reported_and_ignored():
    x, w, b, t = make(20, 64, 300, torch.bfloat16, torch.bfloat16, seed=9)
    cuda_ops.check_device_errors()
    t[2], t[11] = 300, -5
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b)
    grads = torch.autograd.grad(loss, leaves)
    with pytest.raises(RuntimeError, match="target outside the vocabulary"):
        cuda_ops.check_device_errors()
    t[2] = t[11] = -100
    again = linear_cross_entropy(x, w, t, b)
    assert torch.equal(loss, again)
    for a, c in zip(grads, torch.autograd.grad(again, leaves)):
        assert torch.equal(a, c)
    cuda_ops.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_strides_alignment_and_index_types(dtype):
    x, w, b, t = make(130, 96, 400, dtype, dtype, seed=10)
    plain = linear_cross_entropy(x, w, t, b, reduction="none")
    odd = torch.empty(130 * 96 + 1, device=DEV, dtype=dtype)[1:].view(130, 96).copy_(x)           # off any 16-byte boundary
    odd_w = torch.empty(400 * 96 + 1, device=DEV, dtype=dtype)[1:].view(400, 96).copy_(w)
    assert torch.equal(linear_cross_entropy(odd, odd_w, t.int(), b, reduction="none"), plain)
    assert torch.equal(linear_cross_entropy(x.T.contiguous().T, w.T.contiguous().T, t.flip(0).flip(0), b, reduction="none"), plain)
    shaped = linear_cross_entropy(x.view(10, 13, 96), w, t.view(10, 13), b, reduction="none")
    assert shaped.shape == (10, 13) and torch.equal(shaped.flatten(), plain)
    grads = []
    for a, c in ((x, w), (odd, odd_w)):
        a, c = a.detach().requires_grad_(True), c.detach().requires_grad_(True)
        grads.append(torch.autograd.grad(linear_cross_entropy(a, c, t, b), (a, c)))
    for p, q in zip(*grads):
        assert torch.equal(p, q)


def test_only_the_gradients_that_are_asked_for():
    x, w, b, t = make(70, 64, 300, torch.bfloat16, torch.bfloat16, seed=11)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    every = torch.autograd.grad(linear_cross_entropy(x, w, t, b), leaves)
    for i in range(3):
        for j, v in enumerate(leaves):
            v.requires_grad_(i == j)
        (one,) = torch.autograd.grad(linear_cross_entropy(x, w, t, b), leaves[i])
        assert torch.equal(one, every[i])
    for v in leaves:
        v.requires_grad_(True)
    linear_cross_entropy(x, w, t, b).backward()
    assert all(torch.equal(v.grad, e) for v, e in zip(leaves, every))
    with pytest.raises(RuntimeError):                     # the gradient has no gradient of its own
        g = torch.autograd.grad(linear_cross_entropy(x, w, t, b), x, create_graph=True)[0]
        torch.autograd.grad(g.float().sum(), x)


def test_same_bits_every_time_and_on_another_stream():
    x, w, b, t = make(700, 128, 3000, torch.bfloat16, torch.bfloat16, ignored=0.2, seed=12)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]

    def step():
        loss = linear_cross_entropy(x, w, t, b)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    first = step()
    side = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in side:                                    # two streams at a time, each with its own workspace
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                results.append(step())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(p, q) for p, q in zip(first, r))


def test_captured_step_replays_on_new_inputs():
    x, w, b, t = make(300, 128, 1000, torch.bfloat16, torch.bfloat16, ignored=0.2, seed=13)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]

    def step():
        loss = linear_cross_entropy(x, w, t, b)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                    # two graphs over the same leaves
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    x2, w2, b2, t2 = make(300, 128, 1000, torch.bfloat16, torch.bfloat16, ignored=0.4, seed=14)
    with torch.no_grad():
        for old, new in ((x, x2), (w, w2), (b, b2), (t, t2)):
            old.copy_(new)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(out, want))
    cuda_ops.check_device_errors()


def test_the_c_abi_refuses_a_short_workspace_and_writes_only_its_outputs():
    lib = cabi.load()
    x, w, b, t = make(5, 64, 300, torch.bfloat16, torch.bfloat16, seed=15)
    need = lib.grmx_linear_xent_workspace(5, 64, 300, cabi.BF16, 0)
    ws = torch.empty(need, device=DEV, dtype=torch.uint8)
    loss = torch.full((8,), 7.0, device=DEV)
    stats, inv = torch.empty(2, 5, device=DEV), torch.empty(1, device=DEV)
    args = (cabi.ptr(x), cabi.ptr(w), cabi.ptr(b), cabi.ptr(t), -100, cabi.ptr(loss), cabi.ptr(stats), cabi.ptr(inv), 5, 64, 300,
            cabi.BF16, cabi.BF16, cabi.REDUCE_NONE, cabi.ptr(ws))
    assert lib.grmx_linear_xent_fwd(*args, need - 1, cabi.current_stream()) == 1
    assert b"workspace" in lib.grmx_last_error()
    cabi.check(lib.grmx_linear_xent_fwd(*args, need, cabi.current_stream()))
    torch.cuda.synchronize()
    assert torch.equal(loss[:5], linear_cross_entropy(x, w, t, b, reduction="none")) and (loss[5:] == 7.0).all()


def test_norm_and_loss_together_as_the_end_of_a_training_step():
    # the last block's mixing rule and norm, then the vocabulary loss, differentiated through both
    g = torch.Generator(device=DEV).manual_seed(16)
    B, T, H, V = 2, 65, 96, 500
    online, update, gate = (torch.randn(B, T, H, device=DEV, generator=g, requires_grad=True) for _ in range(3))
    scale, lw, lb = ((1 + 0.1 * torch.randn(H, device=DEV, generator=g)).requires_grad_(True) for _ in range(3))
    w = (torch.randn(V, H, device=DEV, generator=g) * 0.2).requires_grad_(True)
    t = torch.randint(0, V, (B, T), device=DEV, generator=g)
    t[:, -9:] = -100
    leaves = (online, update, gate, scale, lw, lb, w)
    loss = linear_cross_entropy(fuse_layer_norm(online, update, lw, lb, gate=gate, scale=scale), w, t)
    grads = torch.autograd.grad(loss, leaves)
    wide = [v.detach().double().requires_grad_(True) for v in leaves]
    o, u, k, s, a, c, m = wide
    mixed = torch.sigmoid(k) * o + (1 - torch.sigmoid(k)) * s * u
    h = torch.nn.functional.layer_norm(mixed, (H,), a, c, 1e-5)
    want = torch.nn.functional.cross_entropy((h @ m.T).flatten(0, 1), t.flatten())
    want_grads = torch.autograd.grad(want, wide)
    # every step is fp32 (2^-24 a rounding, some hundred in a row at worst): 1e-4 of the largest value is far above
    # what they add up to and far below any term that could be missing
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())
    for got, ref in zip(grads, want_grads):
        assert float((got.double() - ref).abs().max()) <= 1e-4 * float(ref.abs().max())


def test_language_model_loss_is_the_cross_entropy_of_its_scores():
    g = torch.Generator(device=DEV).manual_seed(17)
    vocab, B, T = 700, 2, 384
    params = {}
    for name, shape in language_model_parameter_shapes(2, 64, 64, vocab, 64).items():
        v = torch.randn(*shape, device=DEV, generator=g) * (0.1 if len(shape) == 1 else 1.5 / shape[-1] ** 0.5)
        params[name] = (v + 1.0 if "layer_norm.weight" in name else v).bfloat16()
    lm = StackedSegmentMemoryRunner(params, 2, language_model=True, segment_length=128, retrieval_top_k=2,
                                    memory_capacity_segments=4)
    ids = torch.randint(0, vocab, (B, T + 1), device=DEV, generator=g)
    ids, targets = ids[:, :-1].contiguous(), ids[:, 1:].clone()
    targets[1, 300:] = -100
    loss = lm.loss(ids, targets)
    per_token = lm.loss(ids, targets, reduction="none")
    scores, _ = lm.forward(ids)
    lm.vocabulary_projection = False
    y, _ = lm.forward(ids)
    assert torch.equal(per_token, linear_cross_entropy(y, params["output_layer.weight"], targets, params["output_layer.bias"],
                                                       reduction="none"))
    # the forward pass rounds its scores to bf16, half a step each: the target's own and, at most, all others'
    want = torch.nn.functional.cross_entropy(scores.double().flatten(0, 1), targets.flatten(), reduction="none").view(B, T)
    assert ((per_token.double() - want).abs() <= 2 * 2.0 ** -8 * scores.double().abs().amax(-1) + 1e-4).all()
    assert not per_token[1, 300:].any()
    count = int((targets != -100).sum())
    assert abs(float(loss) - float(per_token.double().sum()) / count) <= 1e-6 * float(loss)
    cuda_ops.check_device_errors()


# A last row tile of 1 to 128 rows leaves the second CTA of its pair with boxes that are staged and not sent, behind boxes
# of the group's tile before it that are still on their way: results of more than 148 tiles (74 pairs, two epilogue groups),
# with contractions of one block.
@pytest.mark.parametrize("shape", [(9, 512, 50257), (40, 512, 50257), (64, 512, 50257), (32, 1024, 32800), (64, 331, 50257),
                                   (38500, 64, 50), (19300, 512, 60), (38500, 67, 50)], ids=lambda s: "x".join(map(str, s)))
def test_many_tiles_of_short_contractions_and_a_last_one_half_empty(shape):
    N, D, V = shape
    assert 1 <= max(N, V) % 256 <= 128 and -(-max(N, V) // 256) * -(-D // 256) >= 149
    x, w, b, t = make(N, D, V, torch.bfloat16, torch.float32, ignored=0.1, seed=19)
    t[0] = V - 1
    leaves = [v.requires_grad_(True) for v in (x, w, b)]

    def step():
        return torch.autograd.grad(linear_cross_entropy(x, w, t, b, reduction="sum"), leaves)

    first = step()
    _, _, want_grads, grad_tols = reference(x, w, b, t, torch.ones(N, device=DEV))
    for name, grad in zip("xwb", first):
        within(grad, want_grads[name], grad_tols[name], "gradient of " + name)
    for _ in range(30):
        assert all(torch.equal(p, q) for p, q in zip(first, step()))
    cuda_ops.check_device_errors()


def test_threads_of_different_widths():
    # eight tokens of up to 128 KiB of features in shared memory, from two threads at a time
    inputs = [make(8, D, 64, torch.bfloat16, seed=D) for D in (1536, 2048, 3000, 4096)]
    wants = [linear_cross_entropy(x, w, t, reduction="none") for x, w, _, t in inputs]
    failures = []

    def decode(own):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(3000):
                    x, w, _, t = inputs[own[i % 2]]
                    loss = linear_cross_entropy(x, w, t, reduction="none")
                assert torch.equal(loss, wants[own[1]])
        except Exception as e:  # noqa: BLE001 -- reported by the test's own thread
            failures.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=decode, args=(own,)) for own in ((0, 3), (1, 2), (2, 0), (3, 1))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures[0]


def test_forward_mode_and_function_transforms_are_refused():
    x, w, b, t = make(20, 64, 300, torch.float32, torch.float32, seed=23)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear_cross_entropy(dual, w, t, b)
        with pytest.raises(RuntimeError, match="forward-mode"):
            fuse_layer_norm(dual, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            fuse_layer_norm(x, x, gate=dual)
    linear_cross_entropy(dual, w, t, b)                   # the level is closed: an ordinary tensor again
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: linear_cross_entropy(a, w, t[:5]))(x.view(4, 5, 64))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: linear_cross_entropy(a, w, t))(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: linear_cross_entropy(a, w, t), (x,), (x,))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N", [5, 40], ids=["few tokens", "tiles"])
def test_words_masked_with_the_lowest_value(N, dtype):
    x, w, _, t = make(N, 64, 700, dtype, seed=20)
    low = torch.finfo(dtype).min
    b = torch.zeros(700, device=DEV, dtype=dtype)
    b[256:520] = b[3] = low
    t = torch.where((t >= 256) & (t < 520) | (t == 3), torch.full_like(t, 100), t)
    t[2], t[3] = 300, 3                                  # two tokens whose own word is masked
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b, reduction="none")
    grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    # beside the lowest value the scores vanish: the loss is that value, off by the last bits of fp32 arithmetic
    masked = torch.zeros(N, dtype=torch.bool, device=DEV)
    masked[2:4] = True
    assert ((loss[masked].double() + low).abs() <= 2.0 ** -21 * abs(low)).all()
    size = torch.where(b == low, torch.zeros_like(b), b)  # (the reference's bounds are of the words that are open)
    want, tol, want_grads, grad_tols = reference(x, w, torch.where(b == low, torch.full_like(b, float("-inf")), size), t,
                                                 torch.ones(N, device=DEV))
    within(loss[~masked], want[~masked], tol[~masked], "loss")
    for name, grad in zip("xwb", grads):
        within(grad, want_grads[name], grad_tols[name], "gradient of " + name)


@pytest.mark.parametrize("N", [5, 40], ids=["few tokens", "tiles"])
def test_every_word_masked_with_the_lowest_value(N):
    # all scores are the lowest value: the words are equally likely
    x, w, _, t = make(N, 64, 512, torch.float32, seed=21)
    b = torch.full((512,), torch.finfo(torch.float32).min, device=DEV)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b, reduction="none")
    assert ((loss.double() - 9 * 0.6931471805599453).abs() <= 2.0 ** -20 * 7).all()
    for grad in torch.autograd.grad(loss, leaves, torch.ones_like(loss)):
        assert torch.isfinite(grad).all() and grad.any()


@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("factor", [float("inf"), float("nan")])
def test_ignored_tokens_have_no_gradient_whatever_the_factor_is(reduction, factor):
    x, w, _, t = make(300, 72, 513, torch.bfloat16, ignored=0.3, seed=22)
    x.requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, reduction=reduction)
    (grad,) = torch.autograd.grad(loss, x, torch.tensor(factor, device=DEV))
    assert not grad[t == -100].any() and not torch.isfinite(grad[t != -100]).any()


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (2100, 40, 262400)), (torch.bfloat16, (30011, 300, 18300)), (torch.float32, (700, 40, 262400))],
                         ids=["bf16 cut contraction", "bf16 two column tiles", "fp32 cut contraction"])
def test_pieces_with_a_factor_per_token(dtype, shape):
    N, D, V = shape
    assert 2 * (1 if dtype == torch.bfloat16 else 3) * N * V > 1 << 30       # more than one piece
    x, w, b, t = make(N, D, V, dtype, torch.float32, ignored=0.1, seed=24)
    t[0], t[1] = 0, V - 1
    up = torch.rand(N, device=DEV) + 0.5
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad(linear_cross_entropy(x, w, t, b, reduction="none"), leaves, up)
    rows = torch.arange(0, N, N // 100, device=DEV)
    want, _, want_grads, grad_tols = reference(x[rows], w, b, t[rows], up[rows])
    within(grads[0][rows], want_grads["x"], grad_tols["x"], "gradient of x")
    X, W, B = x.detach().double(), w.detach().double(), b.detach().double()
    lse = torch.cat([torch.logsumexp(torch.addmm(B, X[i:i + 500], W.T), 1) for i in range(0, N, 500)])
    g = torch.where(t != -100, up, torch.zeros_like(up)).double()[:, None]
    e = (D + 16) * 2.0 ** -23 * (X.abs().sum(1) * W.abs().max() + B.abs().max())
    for v0 in (0, V // 2 - 60, V - 120):
        words = torch.arange(v0, v0 + 120, device=DEV)
        p = torch.exp(X @ W[words].T + B[words] - lse[:, None])
        unit = p - (t[:, None] == words).double()
        d = unit * g
        d_tol = g * (p * (2 * e + 2.0 ** -20)[:, None] * 1.01 + HALF_STEP[dtype] * unit.abs())
        # drains of 8 blocks in full precision, the whole contraction in bf16; the tokens times their factor are rounded
        steps = 40 + N * 6 / 512 if dtype == torch.float32 else N + 16
        tol = (d_tol + (steps * 2.0 ** -23 + HALF_STEP[dtype]) * d.abs()).T @ X.abs() + 2 * HALF_STEP[dtype] * (d.T @ X).abs()
        within(grads[1][words], d.T @ X, tol, f"gradient of words from {v0}")
        fine = (d_tol + (40 + N / 32) * 2.0 ** -24 * d.abs()).sum(0)
        within(grads[2][words], d.sum(0), fine + 2 * HALF_STEP[b.dtype] * d.sum(0).abs(), f"bias gradient of words from {v0}")


@pytest.mark.parametrize("shape", [(300, 72, 513), (1500, 300, 5000), (2048, 64, 2048)], ids=lambda s: "x".join(map(str, s)))
def test_full_precision_sums_are_as_short_as_they_are(shape):
    """The accumulator is drained every 8 blocks: 32 accumulations and 8 more roundings around them, then one fp32 addition per
    drain, of which a contraction of `length` has length * 6 / (64 * 8)."""
    N, D, V = shape
    x, w, b, t = make(N, D, V, torch.float32, torch.float32, seed=25)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad(linear_cross_entropy(x, w, t, b, reduction="sum"), leaves)
    X, W = x.detach().double(), w.detach().double()
    y = X @ W.T + b.detach().double()
    e = (D + 16) * 2.0 ** -23 * (X.abs() @ W.abs().T + b.detach().double().abs()).amax(1)
    p = torch.softmax(y, 1)
    d = p.scatter_add(1, t[:, None], torch.full((N, 1), -1.0, device=DEV, dtype=torch.float64))
    d_tol = p * (2 * e + 2.0 ** -20)[:, None] * 1.01 + 2.0 ** -24 * d.abs()
    for name, grad, a, a_tol, other in (("x", grads[0], d, d_tol, W), ("w", grads[1], d.T, d_tol.T, X)):
        steps = 40 + len(other) * 6 / 512
        within(grad, a @ other, (a_tol + steps * 2.0 ** -23 * a.abs()) @ other.abs() + 2.0 ** -23 * (a @ other).abs(), "gradient of " + name)


def test_offsets_beyond_32_bits_of_tokens():
    N, D, V = 4_250_000, 512, 40
    assert N * D > 1 << 31
    x, w, b, t = make(N, D, V, torch.bfloat16, torch.float32, ignored=0.1, seed=26)
    rows = torch.cat([torch.arange(64, device=DEV), torch.arange(N - 300, N, device=DEV)])
    leaves = [v.requires_grad_(True) for v in (x, b)]
    loss = linear_cross_entropy(x, w, t, b, reduction="none")
    dx, db = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    want, tol, want_grads, grad_tols = reference(x[rows], w, b, t[rows], torch.ones(len(rows), device=DEV))
    within(loss[rows], want, tol, "loss")
    within(dx[rows], want_grads["x"], grad_tols["x"], "gradient of x")
    assert torch.isfinite(db).all() and not dx[t == -100].any()


@pytest.mark.parametrize("N", [3, 16], ids=["few tokens", "tiles"])
def test_offsets_beyond_32_bits_of_words(N):
    D, V = 512, 4_250_000
    assert V * D > 1 << 31
    x, w, b, t = make(N, D, V, torch.bfloat16, torch.bfloat16, seed=27)
    t[0], t[1] = V - 1, 4_200_003
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b, reduction="none")
    _, dw, db = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    y = torch.cat([x.double() @ w[i:i + 250_000].detach().double().T + b[i:i + 250_000].double() for i in range(0, V, 250_000)], 1).detach()
    lse = torch.logsumexp(y, 1)
    e = (D + 16) * 2.0 ** -23 * (x.double().abs().sum(1) * float(w.detach().abs().max()) + float(b.detach().abs().max())).detach()
    want = lse - y.gather(1, t[:, None])[:, 0]
    within(loss, want, 2 * e + 2.0 ** -20 * (1 + want.abs()), "loss")
    words = torch.cat([t, torch.arange(V - 300, V, device=DEV)])
    unit = torch.exp(y[:, words] - lse[:, None]) - (t[:, None] == words).double()
    unit_tol = torch.exp(y[:, words] - lse[:, None]) * (2 * e + 2.0 ** -20)[:, None] * 1.01 + 2.0 ** -8 * unit.abs()
    X = x.detach().double()
    # (the tokens' factors are ones: nothing is rounded for them)
    within(dw[words], unit.T @ X, (unit_tol + (N + 16) * 2.0 ** -23 * unit.abs()).T @ X.abs() + 2.0 ** -7 * (unit.T @ X).abs(), "gradient of w")
    within(db[words], unit.sum(0), (unit_tol + 42 * 2.0 ** -24 * unit.abs()).sum(0) + 2.0 ** -7 * unit.sum(0).abs(), "gradient of b")


def test_a_few_wide_tokens_in_a_captured_call():
    x, w, b, t = make(8, 4096, 300, torch.bfloat16, torch.bfloat16, seed=28)
    want = linear_cross_entropy(x, w, t, b, reduction="none")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_cross_entropy(x, w, t, b, reduction="none")
    out.zero_()
    linear_cross_entropy(x[:, :2048], w[:, :2048], t, b)      # a narrower call in between
    graph.replay()
    assert torch.equal(out, want)
