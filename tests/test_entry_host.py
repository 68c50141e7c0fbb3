"""What of the operators at an expert layer's entry needs no GPU: argument checks of the C ABI and of the calls ahead of any device work."""

import ctypes
import inspect
import re

import pytest
import torch

import cabi
import nanoep_amd as ep
from nanoep_amd import norms, router
from nanoep_amd.build import CSRC

BAD, NO_WORKSPACE = 1, 3


def library():
    lib = cabi.lib()
    p, i, i64, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
    lib.nanoep_layer_norm.argtypes = [p, p, p, p, i64, i, f, i, i, p, p, p, p, p]
    lib.nanoep_layer_norm_backward_workspace_bytes.restype = sz
    lib.nanoep_layer_norm_backward_workspace_bytes.argtypes = [i64, i, i]
    lib.nanoep_layer_norm_backward.argtypes = [p, p, p, p, p, p, i64, i, i, i, p, p, p, p, sz, p]
    lib.nanoep_route_topk.argtypes = [p, i64, i, p, p, i64, i, i, i, i, i, i, f, p, p, p]
    lib.nanoep_route_topk_backward.argtypes = [p, p, i64, i, p, i64, i, i, i, i, f, p, p]
    lib.nanoep_balance_loss_workspace_bytes.restype = sz
    lib.nanoep_balance_loss_workspace_bytes.argtypes = [i64, i, i, i64]
    lib.nanoep_balance_loss.argtypes = [p, i64, i, p, p, i64, i, i, i64, i, p, p, p, p, sz, p]
    lib.nanoep_balance_loss_backward.argtypes = [p, p, i64, i, p, p, p, p, i64, i, i, i64, i, p, p]
    return lib


def test_norms_are_refused_before_any_device_work():
    lib, null = library(), None
    norm, backward = lib.nanoep_layer_norm, lib.nanoep_layer_norm_backward
    # no rows are nothing to do
    assert norm(null, null, null, null, 0, 256, 1e-5, 0, 0, null, null, null, null, null) == 0
    # sizes, eps, types
    for tokens, hidden, eps, rows, parameters in ((-1, 256, 0, 0, 0), (1 << 31, 256, 0, 0, 0), (1, 0, 0, 0, 0), (1, 12, 0, 0, 0), (1, 16392, 0, 0, 0),
                                                  (1, 256, -1, 0, 0), (1, 256, float("nan"), 0, 0), (1, 256, 0, 1, 0), (1, 256, 0, 2, 1), (1, 256, 0, 0, 2)):
        assert norm(64, null, 64, null, tokens, hidden, eps, rows, parameters, null, 64, 64, 64, null) == BAD
    # a residual without a place for the sum, a beta without a mean, missing and unaligned pointers
    assert norm(64, 64, 64, null, 1, 256, 0, 0, 0, null, 64, 64, 64, null) == BAD
    assert norm(64, null, 64, 64, 1, 256, 0, 0, 0, null, 64, null, 64, null) == BAD
    assert norm(null, null, 64, null, 1, 256, 0, 0, 0, null, 64, 64, 64, null) == BAD
    assert norm(64, null, 64, null, 1, 256, 0, 0, 0, null, null, 64, 64, null) == BAD
    assert norm(64, null, 64, null, 1, 256, 0, 0, 0, null, 64, 64, null, null) == BAD
    assert norm(72, null, 64, null, 1, 256, 0, 0, 0, null, 64, 64, 64, null) == BAD
    # the gradient: nothing wanted, a beta's without a mean and the other way round, no workspace
    assert backward(64, 64, 64, 64, 64, null, 1, 256, 0, 0, null, null, null, null, 0, null) == BAD
    assert backward(64, 64, 64, null, 64, null, 1, 256, 0, 0, 64, 64, 64, 64, 1 << 20, null) == BAD
    assert backward(64, 64, 64, 64, 64, null, 1, 256, 0, 0, 64, 64, null, 64, 1 << 20, null) == BAD
    assert backward(64, 64, 64, 64, 64, null, 1, 256, 0, 0, 64, null, 64, 64, 1 << 20, null) == BAD
    assert backward(null, 64, 64, 64, 64, null, 1, 256, 0, 0, 64, null, null, null, 0, null) == BAD
    assert backward(64, 64, 64, 64, 64, null, 1, 252, 0, 0, 64, null, null, null, 0, null) == BAD
    needed = lib.nanoep_layer_norm_backward_workspace_bytes(3, 256, 0)
    assert needed >= 2 * 256 * 4 and needed % (2 * 256 * 4) == 0
    assert backward(64, 64, 64, 64, 64, null, 3, 256, 0, 0, 64, 64, 64, 64, needed - 1, null) == NO_WORKSPACE
    assert backward(64, 64, 64, 64, 64, null, 3, 256, 0, 0, 64, 64, 64, null, needed, null) == BAD
    assert lib.nanoep_layer_norm_backward_workspace_bytes(0, 256, 0) == 0 and lib.nanoep_layer_norm_backward_workspace_bytes(-1, 256, 0) == 0
    # what it holds does not grow with the rows beyond the device's size
    assert lib.nanoep_layer_norm_backward_workspace_bytes(1 << 30, 256, 0) <= 2048 * 2 * 256 * 4


def test_routers_are_refused_before_any_device_work():
    lib, null = library(), None
    route, backward = lib.nanoep_route_topk, lib.nanoep_route_topk_backward

    def routed(stride=64, kind=0, tokens=1, experts=64, topk=8, groups=1, topk_groups=1, scoring=0, logits=64, ids=64):
        return route(logits, stride, kind, null, null, tokens, experts, topk, groups, topk_groups, scoring, 1, 1.0, ids, 64, null)

    def returned(stride=64, kind=0, tokens=1, experts=64, topk=8, scoring=0, grad=64, ids=64):
        return backward(grad, 64, stride, kind, ids, tokens, experts, topk, scoring, 1, 1.0, 64, null)

    assert routed(tokens=0, logits=null) == 0 and returned(tokens=0, grad=null) == 0
    for wrong in ({"stride": 63}, {"stride": (1 << 31) + 1}, {"kind": 2}, {"tokens": -1}, {"tokens": 1 << 26}, {"experts": 0}, {"experts": 4097, "stride": 5000}, {"topk": 0},
                  {"topk": 33}, {"scoring": 2}, {"ids": null}):
        assert routed(**wrong) == BAD and returned(**wrong) == BAD, wrong
    for wrong in ({"topk": 9, "experts": 8}, {"groups": 0}, {"groups": 3}, {"groups": 65, "experts": 65, "stride": 65}, {"groups": 8, "topk_groups": 0},
                  {"groups": 8, "topk_groups": 9}, {"groups": 16, "topk_groups": 1}, {"logits": null}):
        assert routed(**wrong) == BAD, wrong
    assert returned(grad=null) == BAD


def test_balance_losses_are_refused_before_any_device_work():
    lib, null = library(), None

    def lost(stride=64, kind=0, tokens=1, experts=64, topk=8, sequences=1, offsets=null, scoring=0, ids=64, loss=64, workspace=null, size=0):
        return lib.nanoep_balance_loss(64, stride, kind, ids, offsets, tokens, experts, topk, sequences, scoring, loss, 64, 64, workspace, size, null)

    def returned(stride=64, kind=0, tokens=1, experts=64, topk=8, sequences=1, offsets=null, scoring=0, ids=64, loss=64):
        return lib.nanoep_balance_loss_backward(loss, 64, stride, kind, ids, 64, 64, offsets, tokens, experts, topk, sequences, scoring, 64, null)

    assert returned(tokens=0, loss=null) == 0
    for wrong in ({"stride": 63}, {"kind": 2}, {"tokens": -1}, {"tokens": 1 << 26}, {"experts": 0}, {"experts": 4097, "stride": 5000}, {"topk": 0}, {"topk": 33},
                  {"scoring": 2}, {"ids": null}, {"sequences": 0}, {"sequences": 2}, {"sequences": 1 << 31, "offsets": 64}, {"loss": null}):
        assert lost(**wrong) == BAD and returned(**wrong) == BAD, wrong
    needed = lib.nanoep_balance_loss_workspace_bytes(100_000, 64, 8, 1)
    assert needed > 0 and lib.nanoep_balance_loss_workspace_bytes(10, 64, 8, 1) == 0 and lib.nanoep_balance_loss_workspace_bytes(10, 0, 8, 1) == 0
    assert lost(tokens=100_000, workspace=64, size=needed - 1) == NO_WORKSPACE
    assert lost(tokens=100_000, workspace=null, size=needed) == BAD and lost(tokens=100_000, workspace=72, size=needed) == BAD


def test_cpu_tensors_are_refused():
    x, gamma, stat = torch.zeros(2, 256), torch.ones(256), torch.ones(2)
    logits, ids, weights = torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int64), torch.ones(2, 1)
    counts, tokens = torch.zeros(8, dtype=torch.int64), torch.zeros((), dtype=torch.int64)
    for call in (lambda: ep.layer_norm(x, gamma), lambda: ep.rms_norm(x, gamma), lambda: ep.layer_norm_backward(x, x, gamma, stat, stat),
                 lambda: ep.rms_norm_backward(x, x, gamma, stat), lambda: ep.route_topk(logits, 1), lambda: ep.route_topk_backward(weights, logits, ids),
                 lambda: ep.balance_loss(logits, ids), lambda: ep.balance_loss_backward(stat[0], logits, ids, counts, tokens),
                 lambda: ep.layer_norm(x.requires_grad_(), gamma), lambda: ep.route_topk(logits.requires_grad_(), 1), lambda: ep.balance_loss(logits, ids)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()


def test_scorings_are_named():
    logits, ids, weights = torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int64), torch.ones(2, 1)
    for call in (lambda: ep.route_topk(logits, 1, scoring="relu"), lambda: ep.route_topk_backward(weights, logits, ids, scoring=0),
                 lambda: ep.balance_loss(logits, ids, scoring=None)):
        with pytest.raises(ValueError, match="scoring must be one of softmax, sigmoid"):
            call()


def test_every_function_that_the_entry_binds_is_called():
    bound = set(re.findall(r'module\.def\("(\w+)"', (CSRC / "nanoep_entry.cpp").read_text()))
    called = set(re.findall(r"(?:load_extension\(\)|extension)\.(\w+)\(", inspect.getsource(norms) + inspect.getsource(router)))
    assert bound == called
