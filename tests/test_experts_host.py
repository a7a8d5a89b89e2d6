"""The host's half of the operators of a layer of experts, without a GPU: what the library refuses before it touches the device."""
import pytest
import torch

import apt_b200
from apt_b200 import _lib

lib = _lib.lib
P = 1 << 20      # an address that nothing here reads


@pytest.mark.parametrize("experts,k,groups,top,best,text", [
    (0, 1, 1, 1, 1, b"0 experts"), (1025, 1, 1, 1, 1, b"1025 experts"), (8, 9, 1, 1, 1, b"9 of 8"), (128, 65, 1, 1, 1, b"65 of 128"), (8, 0, 1, 1, 1, b"0 of 8"),
    (8, 2, 3, 1, 1, b"3 groups"), (64, 2, 64, 1, 1, b"64 groups"), (8, 2, 4, 5, 1, b"5 of 4"), (8, 5, 4, 2, 1, b"2 of 4"), (8, 2, 4, 2, 0, b"not 0")])
def test_a_router_is_refused(experts, k, groups, top, best, text):
    got = lib.apt_route_experts(_lib.F32, P, 4, experts, k, _lib.SCORE_SOFTMAX, None, groups, top, best, 1, 1.0, P, P, None)
    assert got == _lib.APT_ERR_BAD_ARG and text in lib.apt_last_error()


def test_other_arguments_are_refused():
    assert lib.apt_route_experts(7, P, 4, 8, 2, 0, None, 1, 1, 1, 1, 1.0, P, P, None) == _lib.APT_ERR_BAD_ARG
    assert lib.apt_route_experts(_lib.F32, P, 4, 8, 2, 5, None, 1, 1, 1, 1, 1.0, P, P, None) == _lib.APT_ERR_BAD_ARG
    assert lib.apt_route_experts(_lib.F32, None, 4, 8, 2, 0, None, 1, 1, 1, 1, 1.0, P, P, None) == _lib.APT_ERR_BAD_ARG
    assert lib.apt_route_experts_backward(_lib.F32, P, 4, 8, 2, 0, 1, 1.0, P, None, P, None) == _lib.APT_ERR_BAD_ARG
    assert lib.apt_expert_rows(P, 2 ** 30, 64, P, 2, 8, P, P, P, None, 0, P, None) == _lib.APT_ERR_BAD_ARG
    assert lib.apt_expert_rows(P, 8000, 64, P, 2, 8, P, P, P, None, 0, P, None) == _lib.APT_ERR_BAD_ARG and b"workspace" in lib.apt_last_error()
    assert lib.apt_expert_rows(P, 4, 63, P, 2, 8, P, P, P, None, 0, P, None) == _lib.APT_ERR_BAD_ARG
    assert lib.apt_expert_sum(_lib.F32, P, 2 ** 30, 8, 2, P, P, P, P, None) == _lib.APT_ERR_BAD_ARG
    assert lib.apt_expert_sum_backward(_lib.F32, P, 4, 8, 2, None, P, P, P, P, P, None) == _lib.APT_ERR_BAD_ARG


def test_few_pairs_take_no_workspace():
    assert lib.apt_expert_rows_workspace_bytes(4096, 1024) == 0
    for pairs, experts in ((4097, 1), (1, 1025), (10 ** 6, 64), (10 ** 8, 4096)):
        assert lib.apt_expert_rows_workspace_bytes(pairs, experts) == (experts + 1) * (-(-pairs // 1024) + 1) * 4


def test_cpu_tensors_are_refused():
    z = torch.zeros((4, 8))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        apt_b200.route_experts(z, 2)
    with pytest.raises(RuntimeError, match="unknown score"):
        apt_b200.route_experts(z, 2, "tanh")


def test_more_experts_a_row_than_can_be_counted_are_refused():
    """Pairs are counted in steps beyond the last one: the same limit as that of expert_rows."""
    for k in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 1024):
        for got in (lib.apt_expert_sum(_lib.F32, P, 1, 8, k, P, P, P, P, None), lib.apt_expert_sum_backward(_lib.F32, P, 1, 8, k, P, P, P, P, P, P, None),
                    lib.apt_expert_rows(P, 1, 64, P, k, 8, P, P, P, P, 2 ** 40, P, None)):
            assert got == _lib.APT_ERR_BAD_ARG and b"experts each" in lib.apt_last_error()
