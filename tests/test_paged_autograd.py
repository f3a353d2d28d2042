"""What the paged-cache operators owe to autograd: they record nothing, so whatever asks for a derivative is refused, and what they write
is known to have been written.  On the CPU a call that is not refused for that is refused for its device."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from vits_amd import ops


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def calls():
    q, cache, v = torch.zeros(2, 4, 64), torch.zeros(5, 2, 2, 16, 64), torch.zeros(2, 2, 64)
    k_cache, v_cache = cache[:, 0].clone(), cache[:, 1].clone()
    attention = dict(q=q, k_cache=k_cache, v_cache=v_cache, table=torch.zeros(3, 4, dtype=torch.int32), request=i32(0, 1), position=i32(3, 4),
                     out=torch.zeros(2, 4, 64), lse=torch.zeros(2, 4))
    rotary = dict(q=q, k=v, v=v.clone(), k_cache=k_cache, v_cache=v_cache, slot=torch.arange(2), freq=ops.rotary_frequencies(64, device="cpu"),
                  position=i32(3, 4), out=torch.zeros(2, 4, 64))
    return [(ops.paged_attention, attention, name) for name in ("q", "k_cache", "v_cache", "out", "lse")] + \
           [(ops.rotary_store, rotary, name) for name in ("q", "k", "v", "k_cache", "v_cache", "freq", "out")]


@pytest.mark.parametrize("call,args,name", calls(), ids=lambda x: getattr(x, "__name__", x if isinstance(x, str) else ""))
def test_gradients_are_refused(call, args, name):
    asks = {**args, name: args[name].clone().requires_grad_()}
    with pytest.raises(ValueError, match="gradient"):
        call(**asks)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        call(**asks)


@pytest.mark.parametrize("call,args,name", calls(), ids=lambda x: getattr(x, "__name__", x if isinstance(x, str) else ""))
def test_tangents_are_refused(call, args, name):
    with forward_ad.dual_level():
        dual = {**args, name: forward_ad.make_dual(args[name], torch.ones_like(args[name]))}
        with pytest.raises(ValueError, match="tangent"):
            call(**dual)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):       # which switches off gradients alone
            call(**dual)
        with pytest.raises(ValueError, match="GPU"):
            call(**args)
    with pytest.raises(ValueError, match="GPU"):
        call(**args)
