"""CPU tests of the training operators' argument checks: what is refused before anything touches a device."""

import pytest
import torch

from rnn_with_grm_b200 import cabi
from rnn_with_grm_b200.build import build_all
from rnn_with_grm_b200.fusion import fuse_layer_norm
from rnn_with_grm_b200.loss import linear_cross_entropy
from rnn_with_grm_b200.segment_memory import StackedSegmentMemoryRunner, language_model_parameter_shapes


@pytest.fixture(scope="module")
def lib():
    build_all()
    return cabi.load()


def test_loss_entry_points_refuse_bad_arguments(lib):
    ws = lib.grmx_linear_xent_workspace
    assert ws(0, 64, 100, cabi.BF16, 0) == 0 and ws(0, 64, 100, cabi.BF16, 1) == 0
    assert ws(10, 64, 100, cabi.F16, 0) == -1 and b"dtype" in lib.grmx_last_error()
    assert ws(-1, 64, 100, cabi.BF16, 0) == -1 and ws(10, 0, 100, cabi.BF16, 0) == -1 and ws(10, 64, 0, cabi.BF16, 1) == -1
    assert ws(1 << 29, 64, 100, cabi.BF16, 0) == -1 and b"tile coordinates" in lib.grmx_last_error()
    assert ws(1 << 28, 64, 1 << 28, cabi.BF16, 0) == -1 and b"too many tiles" in lib.grmx_last_error()
    # the gradient of the scores takes at most 1 GiB, whatever the vocabulary
    assert ws(65536, 512, 32768, cabi.BF16, 1) < (1 << 30) + (1 << 30)
    fwd = lib.grmx_linear_xent_fwd
    some = 256                                            # never dereferenced: refused first
    assert fwd(None, None, None, None, -100, None, None, None, 4, 64, 100, cabi.BF16, cabi.BF16, 2, None, 0, None) == 1
    assert b"NULL" in lib.grmx_last_error()
    assert fwd(some, some, None, some, -100, some, some, some, 4, 64, 100, cabi.BF16, cabi.BF16, 3, some, 1 << 30, None) == 1
    assert b"reduction" in lib.grmx_last_error()
    assert fwd(some, some, some, some, -100, some, some, some, 4, 64, 100, cabi.BF16, cabi.F16, 2, some, 1 << 30, None) == 1
    assert b"bias" in lib.grmx_last_error()
    assert fwd(some, some, None, some, -100, some, some, some, 0, 64, 100, cabi.BF16, cabi.BF16, 2, some, 1 << 30, None) == 1
    assert fwd(some, some, None, some, -100, some, some, some, 4, 64, 100, cabi.BF16, cabi.BF16, 2, some, 8, None) == 1
    assert b"workspace" in lib.grmx_last_error()
    assert fwd(some, some, None, some, -100, some, some, some, 4, 64, 100, cabi.BF16, cabi.BF16, 2, some + 16, 1 << 30, None) == 1
    assert b"aligned" in lib.grmx_last_error()
    bwd = lib.grmx_linear_xent_bwd
    assert bwd(None, None, None, None, None, -100, None, None, some, None, None, 4, 64, 100, 1, 1, 2, None, 0, None) == 1
    assert b"NULL" in lib.grmx_last_error()
    assert bwd(some, some, some, None, some, -100, some, some, some, None, None, 4, 64, 100, 1, 1, 2, some, 8, None) == 1
    assert b"workspace" in lib.grmx_last_error()
    # nothing asked for: nothing to do
    assert bwd(None, None, None, None, None, -100, None, None, None, None, None, 4, 64, 100, 1, 1, 2, None, 0, None) == 0


def test_fuse_norm_entry_points_refuse_bad_arguments(lib):
    assert lib.grmx_fuse_norm_workspace(0, 64) == 0 and lib.grmx_fuse_norm_workspace(10, 0) == -1
    assert lib.grmx_fuse_norm_workspace(10, 8193) == -1 and b"at most 8192" in lib.grmx_last_error()
    fwd, some = lib.grmx_fuse_norm_fwd, 256
    assert fwd(*[None] * 6, 1e-5, None, None, None, 0, 64, cabi.BF16, cabi.BF16, None) == 0
    assert fwd(*[None] * 6, 1e-5, None, None, None, 4, 64, cabi.BF16, cabi.BF16, None) == 1
    assert fwd(some, some, None, None, None, None, 1e-5, some, None, None, 4, 64, cabi.F16, cabi.F16, None) == 1
    assert fwd(some, some, None, None, None, None, 1e-5, some, None, None, 4, 64, cabi.F32, cabi.BF16, None) == 1
    assert b"parameters" in lib.grmx_last_error()
    assert fwd(some, some, None, None, None, None, 1e-5, some, None, None, 4, 9000, cabi.F32, cabi.F32, None) == 2
    bwd = lib.grmx_fuse_norm_bwd
    tail = (4, 64, cabi.F32, cabi.F32)
    assert bwd(some, None, some, some, None, None, None, some, some, some, some, None, None, None, *tail, None, 0, None) == 1
    assert b"no gate" in lib.grmx_last_error()
    assert bwd(some, None, some, some, None, None, None, some, some, some, None, some, None, None, *tail, None, 0, None) == 1
    assert b"no scale" in lib.grmx_last_error()
    assert bwd(None, None, some, some, None, None, None, some, some, some, None, None, None, None, *tail, None, 0, None) == 1
    assert b"neither" in lib.grmx_last_error()
    assert bwd(some, None, some, some, None, None, some, some, some, some, None, None, some, None, *tail, None, 0, None) == 1
    assert b"workspace" in lib.grmx_last_error()


def test_python_entry_points_refuse_host_tensors_and_bad_names(lib):
    x, w, t = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA device"):
        linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(RuntimeError, match="CUDA device"):
        fuse_layer_norm(x, x)
    with pytest.raises(NotImplementedError):              # no CPU kernel is registered with the dispatcher
        torch.ops.grmx.linear_xent_fwd(x, w, t, None, -100, 0)
    with pytest.raises(NotImplementedError):
        torch.ops.grmx.fuse_norm_fwd(x, x, None, None, None, None, 1e-5, False, False)


def test_language_model_loss_checks_its_arguments(lib):
    shapes = language_model_parameter_shapes(1, 64, 64, 100, 64)
    kwargs = dict(segment_length=128, retrieval_top_k=2, memory_capacity_segments=4)
    lm = StackedSegmentMemoryRunner({k: torch.zeros(s) for k, s in shapes.items()}, 1, language_model=True, **kwargs)
    ids = torch.zeros(2, 128, dtype=torch.long)
    with pytest.raises(ValueError, match="shape"):
        lm.loss(ids, ids[:, :-1])
    body = {k[len("grm_rnn."):]: torch.zeros(s) for k, s in shapes.items() if k.startswith("grm_rnn.")}
    with pytest.raises(ValueError, match="language"):
        StackedSegmentMemoryRunner(body, 1, **kwargs).loss(ids, ids)


def test_fuse_norm_refuses_row_statistics_off_their_pairs(lib):
    some, tail = 256, (4, 64, cabi.F32, cabi.F32)
    for off in (260, 258, 257):
        assert lib.grmx_fuse_norm_fwd(some, some, None, None, None, None, 1e-5, some, None, off, *tail, None) == 1
        assert b"row_stats must be 8-byte aligned" in lib.grmx_last_error()
        assert lib.grmx_fuse_norm_bwd(some, None, some, some, None, None, None, off, some, some, None, None, None, None, *tail,
                                      None, 0, None) == 1
        assert b"row_stats must be 8-byte aligned" in lib.grmx_last_error()


def test_tangents_are_refused_before_anything_else(lib):
    # (the extension's entry points themselves, which look at tangents before they look at devices)
    from torch.autograd import forward_ad

    from rnn_with_grm_b200 import cuda_ops

    cuda_ops._require_extension("test")
    module = cuda_ops._Extension.module
    x, w, t, v = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.long), torch.zeros(8)
    b = torch.zeros(10)
    with forward_ad.dual_level():
        def dual(a):
            return forward_ad.make_dual(a, torch.ones_like(a))

        for args in ((dual(x), w, t, b), (x, dual(w), t, b), (x, w, t, dual(b))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                module.linear_cross_entropy(*args, -100, 2)
        for i in range(6):
            args = [x, x, v, v, x, v]
            args[i] = dual(args[i])
            with pytest.raises(RuntimeError, match="forward-mode"):
                module.fuse_layer_norm(*args, 1e-5, False)
