"""GPU: the paged cache's operators have no derivatives and say so."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from blockedattention_b200 import blockPagedAppend, blockPagedAttention
from test_paged_gpu import F16, make

pytestmark = pytest.mark.gpu
OPERANDS = ("q", "kCache", "vCache")


def attention_call():
    q, k, v, table, n = make([300, 17], 2, 2, 64, 16, F16)
    return dict(q=q, kCache=k, vCache=v, pageTable=table, lengths=n)


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("name", OPERANDS)
def test_attention_refuses_gradients(cuda_device, name, lse):
    a = attention_call()
    want = blockPagedAttention(**a)
    wants = {**a, name: a[name].clone().requires_grad_()}
    with pytest.raises(RuntimeError, match="forward only"):
        blockPagedAttention(**wants, return_lse=lse)
    with torch.no_grad():
        out = blockPagedAttention(**wants, return_lse=lse)
    assert torch.equal(out[0] if lse else out, want)
    assert torch.equal(blockPagedAttention(**{**wants, name: wants[name].detach()}), want)
    with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        blockPagedAttention(**{**a, name: fwad.make_dual(a[name], torch.ones_like(a[name]))}, return_lse=lse)


@pytest.mark.parametrize("name", ("k", "v", "kCache", "vCache"))
def test_append_refuses_gradients(cuda_device, name):
    c = torch.zeros((2, 1, 16, 64), device="cuda")
    a = dict(k=torch.ones((1, 1, 64), device="cuda"), v=torch.ones((1, 1, 64), device="cuda"), kCache=c, vCache=c.clone(), slots=torch.tensor([3], device="cuda"))
    wants = {**a, name: a[name].clone().requires_grad_()}
    with pytest.raises(RuntimeError, match="gradient"):
        blockPagedAppend(**wants)
    assert (a["kCache"] == 0).all() and (a["vCache"] == 0).all()
    with torch.no_grad():
        blockPagedAppend(**wants)
    assert (wants["kCache"][0, 0, 3] == 1).all() and (wants["vCache"][0, 0, 3] == 1).all()


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", OPERANDS)
def test_traces_refuse_gradients(cuda_device, name):
    a = attention_call()
    plain, wants = tuple(a.values()), tuple({**a, name: a[name].clone().requires_grad_()}.values())
    call = lambda *x: blockPagedAttention(*x, 0.125)
    with pytest.raises(RuntimeError, match="forward only"):
        torch.jit.trace(call, wants, check_trace=False)
    traced = torch.jit.trace(call, plain, check_trace=False)
    assert torch.equal(traced(*plain), call(*plain))
    with pytest.raises(RuntimeError, match="forward only"):   # a replay as well
        traced(*wants)
    with torch.no_grad():
        traced = torch.jit.trace(call, wants, check_trace=False)
        assert torch.equal(traced(*wants), call(*plain))
    got = traced(*wants)   # recorded without gradients: as detached tensors
    assert torch.equal(got, call(*plain)) and not got.requires_grad
