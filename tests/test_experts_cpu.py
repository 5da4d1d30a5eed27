"""Argument checks of the expert and 8-bit entry points, which run on the host before any launch."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)


def _raises(call, match=None, exc=ValueError):
    from sklearn_numba_dpex_b200 import _cabi

    with pytest.raises(exc, match=match):
        _cabi.check(call(_cabi.lib))


def test_route_checks():
    def route(dtype=0, n=4, e=8, k=2, flags=0, groups=1, topk_groups=1, best=1, logits=P):
        return lambda lib: lib.kmb_route_topk(dtype, logits, None, n, e, k, flags, groups, topk_groups, best, 1.0, P, P, None)

    _raises(route(dtype=1), "dtype")                       # KMB_F64
    _raises(route(dtype=7), "dtype")
    _raises(route(e=1025), "number of experts")
    _raises(route(e=0), "number of experts")
    for k in (0, 9, 33):
        _raises(route(k=k), "k must be")
    _raises(route(e=64, k=33), "k must be")
    _raises(route(n=-1), "sizes")
    _raises(route(flags=4), "flag")
    _raises(route(groups=3), "groups")
    _raises(route(e=64, groups=64), "groups")
    _raises(route(groups=4, topk_groups=5), "topk_groups")
    _raises(route(groups=4, topk_groups=0), "topk_groups")
    _raises(route(groups=4, k=3), "search space")
    _raises(route(groups=4, topk_groups=2, best=3), "group_best")
    _raises(route(groups=8, topk_groups=2, best=2), "group_best")
    _raises(route(logits=None), "NULL")

    def grad(dtype=0, e=8, k=2, flags=0, logits=P):
        return lambda lib: lib.kmb_route_topk_grad(dtype, logits, P, P, 4, e, k, flags, 1.0, P, None)

    _raises(grad(dtype=1), "dtype")
    _raises(grad(e=1025), "number of experts")
    _raises(grad(k=9), "k must be")
    _raises(grad(flags=8), "flag")
    _raises(grad(logits=None), "NULL")


def test_slots_and_combine_checks():
    from sklearn_numba_dpex_b200 import _cabi

    lib = _cabi.lib
    _raises(lambda l: l.kmb_expert_slots(P, 4, 2, 1025, P, P, P, None, 0, None), "number of experts")
    _raises(lambda l: l.kmb_expert_slots(P, 4, 0, 8, P, P, P, None, 0, None), "sizes")
    _raises(lambda l: l.kmb_expert_slots(P, 1 << 30, 2, 8, P, P, P, None, 0, None), "2\\^31")
    _raises(lambda l: l.kmb_expert_slots(None, 4, 2, 8, P, P, P, None, 0, None), "NULL")
    assert lib.kmb_expert_slots_workspace_bytes(64, 8, 256) == 0
    need = lib.kmb_expert_slots_workspace_bytes(5000, 8, 256)
    assert need > 0
    _raises(lambda l: l.kmb_expert_slots(P, 5000, 8, 256, P, P, P, P, need - 1, None), "workspace", _cabi.KmbError)
    _raises(lambda l: l.kmb_combine_experts(1, P, 4, P, P, 4, 2, 8, P, None), "dtype")
    _raises(lambda l: l.kmb_combine_experts(0, P, 4, P, P, 4, 0, 8, P, None), "sizes")
    _raises(lambda l: l.kmb_combine_experts(0, None, 4, P, P, 4, 2, 8, P, None), "NULL")
    _raises(lambda l: l.kmb_combine_experts(0, P, 4, P, P, 4, 2, 1 << 30, P, None), "2\\^30")
    _raises(lambda l: l.kmb_combine_experts_grad(0, P, 4, P, P, P, 4, 2, 1 << 30, P, P, P, 1 << 20, None), "2\\^30")
    need = lib.kmb_combine_experts_grad_workspace_bytes(100)
    _raises(lambda l: l.kmb_combine_experts_grad(0, P, 100, P, P, P, 4, 2, 8, P, P, P, need - 1, None), "workspace",
            _cabi.KmbError)
    _raises(lambda l: l.kmb_combine_experts_grad(0, P, 100, P, P, P, 1 << 30, 2, 8, P, P, P, need, None), "2\\^31")


def test_int8_checks():
    def product(out=0, a=P, lda=32, ldb=32, groups=1, offsets=None, m=4, n=8, d=32):
        return lambda lib: lib.kmb_int8_matmul(out, a, lda, P, P, ldb, P, None, offsets, groups, P, m, n, d, None)

    _raises(product(out=1), "out_dtype")
    _raises(product(d=131072, lda=131072, ldb=131072), "131071")
    _raises(product(lda=40), "pitches")
    _raises(product(lda=16), "pitches")
    _raises(product(ldb=16), "pitches")
    _raises(product(a=ctypes.c_void_p(264)), "aligned")
    _raises(product(groups=2), "groups")
    _raises(product(groups=1025, offsets=P), "groups")
    _raises(product(groups=1024, offsets=P, n=1 << 22), "groups \\* n")
    _raises(product(a=None), "NULL")
    _raises(product(n=0), "sizes")
    _raises(lambda l: l.kmb_quantize_rows(1, P, 4, 8, None, 4, P, 16, P, None), "dtype")
    _raises(lambda l: l.kmb_quantize_rows(0, P, 4, 8, None, 5, P, 16, P, None), "m must be n")
    _raises(lambda l: l.kmb_quantize_rows(0, P, 4, 1 << 30, None, 4, P, 1 << 30, P, None), "2\\^30")
    _raises(lambda l: l.kmb_quantize_rows(0, P, 4, 8, None, 4, P, 8, P, None), "pitch")
    _raises(lambda l: l.kmb_quantize_rows(0, P, 4, 20, None, 4, P, 16, P, None), "pitch")
    _raises(lambda l: l.kmb_quantize_rows(0, None, 4, 8, None, 4, P, 16, P, None), "NULL")


def test_host_tensors_are_refused():
    from sklearn_numba_dpex_b200 import common

    x = torch.zeros(4, 8)
    i32, q = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 8, dtype=torch.int8)
    for call in (lambda: common.route_topk(x, 2), lambda: common.route_topk_grad(x, i32, x[:, :2]),
                 lambda: common.expert_slots(i32, 8), lambda: common.combine_experts(x, i32, x[:, :2]),
                 lambda: common.combine_experts_grad(x, i32, x[:, :2], x), lambda: common.quantize_rows(x),
                 lambda: common.int8_matmul(q, x[:, 0], q, x[:, 0])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def test_number_of_choices():
    """Up to 2^31 - 4097 choices in all, however many a token has."""
    for n, k in (((1 << 31) - 4096, 1), (1 << 29, 4), (1, (1 << 31) - 4096), (3, 715826550)):
        _raises(lambda l: l.kmb_expert_slots(P, n, k, 8, P, P, P, P, 1 << 40, None), "below 2\\^31 - 4096")
        _raises(lambda l: l.kmb_combine_experts_grad(0, P, 100, P, P, P, n, k, 8, P, P, P, 1 << 20, None), "below 2\\^31 - 4096")
    from sklearn_numba_dpex_b200 import _cabi

    for n, k in (((1 << 31) - 4097, 1), (1, 600000), (1, (1 << 31) - 4097)):       # the next thing they lack is a workspace
        if _cabi.lib.kmb_expert_slots_workspace_bytes(n, k, 8):
            _raises(lambda l: l.kmb_expert_slots(P, n, k, 8, P, P, P, None, 0, None), "workspace", _cabi.KmbError)
        _raises(lambda l: l.kmb_combine_experts_grad(0, P, 100, P, P, P, n, k, 8, P, P, None, 0, None), "workspace", _cabi.KmbError)
