"""Copies of a packed matrix (ops.Packed8): a copied module or a saved state holds packed weights and checkpoints like any tensor, so the addresses that
the kernels get have to be those of the copy's own tensors."""
import copy
import io
import pickle

import pytest
import torch

from speedplusbaseline_amd import ops


def saved(P):
    f = io.BytesIO()
    torch.save(P, f)
    f.seek(0)
    return torch.load(f, weights_only=False)          # a file of this test's own


COPIES = [copy.deepcopy, lambda P: pickle.loads(pickle.dumps(P)), saved]


def one(rows, K, block_rows, device, separate):
    P = ops.Packed8.empty(rows, K, block_rows, device)
    P.codes.copy_((torch.arange(P.codes.numel(), device=device) % 127).to(torch.uint8).view_as(P.codes))
    P.scales.copy_((120 + torch.arange(P.scales.numel(), device=device) % 9).to(torch.uint8).view_as(P.scales))
    return ops.Packed8(P.codes.clone(), P.scales.clone(), K, block_rows) if separate else P


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("how", COPIES, ids=["deepcopy", "pickle", "save"])
def test_copies_have_their_own_addresses(how, separate):
    P = one(5, 300, 1, "cpu", separate)
    Q = how(P)
    assert Q.shape == P.shape and (Q.K, Q.block_rows) == (P.K, P.block_rows)
    assert torch.equal(Q.codes, P.codes) and torch.equal(Q.scales, P.scales) and Q.device == P.device
    assert Q.codes.data_ptr() != P.codes.data_ptr()
    for R in (P, Q, copy.copy(P)):
        assert R._at() == (R.codes.data_ptr(), R.scales.data_ptr())
    Q.codes.zero_()
    assert P.codes.any()


def test_a_callers_tensors_with_other_storage():
    """what Module.to does to a parameter: the tensor object stays, its storage is another one"""
    P = one(5, 300, 1, "cpu", True)
    codes, scales = P._own
    codes.data = codes.data.clone()
    assert P._at() == (codes.data_ptr(), scales.data_ptr())
    ops.Packed8._check(P)
    for wrong in (torch.zeros(4, 384, dtype=torch.uint8), torch.zeros(5, 384, dtype=torch.int8), torch.zeros(384, 5, dtype=torch.uint8).t()):
        codes.data = wrong
        with pytest.raises(RuntimeError):
            P._check()


@pytest.mark.gpu
def test_products_after_other_storage(device):
    A, B = one(37, 300, 1, "cuda", True), one(130, 300, 128, "cuda", False)
    want = ops.gemm8(A, B)
    codes = A._own[0]
    old, codes.data = codes.data, codes.data.clone()
    old.zero_()
    assert torch.equal(ops.gemm8(A, B), want)
    codes.data = codes.data.cpu()
    with pytest.raises(RuntimeError):
        ops.gemm8(A, B)


@pytest.mark.gpu
@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("how", COPIES, ids=["deepcopy", "pickle", "save"])
def test_products_of_copies(device, how, separate):
    """every reader of a packed operand, on copies whose original holds something else by then"""
    from speedplusbaseline_amd import _lib as L
    A, B = one(37, 300, 1, "cuda", separate), one(130, 300, 128, "cuda", separate)
    G = torch.randn(37, 24, device="cuda")
    D = torch.randn(37, 300, device="cuda")
    every = lambda a, b: (ops.gemm8(a, b, dtype=torch.float32), ops.gemm8(a, b), ops.gemm8_wgrad(G, a), ops.dequant8(a), ops.dequant8(b),    # noqa: E731
                          ops.act8_bwd(D, a, L.ACT_SILU))
    want = every(A, B)
    a, b = how(A), how(B)
    A.codes.zero_(), B.codes.zero_(), A.scales.fill_(127), B.scales.fill_(127)
    assert all(torch.equal(x, y) for x, y in zip(every(a, b), want))
    assert not ops.gemm8(A, B).any()
