"""paged_attention has no backward pass: it says so where a gradient is asked for."""
import pytest
import torch

from conftest import load_mod
from test_gpu_paged import make, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("which", ["q", "sinks", "kp", "vp"])
def test_backward_raises(fa, gpu, monkeypatch, binding, which):
    if not binding:
        monkeypatch.setattr(load_mod("_ops"), "_BINDING", None)
    c = make(41, "bf16", "bf16", 64, 4, 2, 16, "hnd", (40, 9), nan=False)
    t = {n: c[n].to(gpu) for n in ("q", "kp", "vp", "table", "lens", "sinks")}
    run = lambda: fa.paged_attention(t["q"], t["kp"], t["vp"], t["table"], t["lens"], sinks=t["sinks"])
    want = run()
    assert not want.requires_grad
    t[which].requires_grad_()
    o = run()
    assert o.requires_grad
    same(o.detach(), want)
    with pytest.raises(NotImplementedError, match="no backward"):
        (o.float() * 2).sum().backward()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            o = run()
        assert not o.requires_grad
        same(o, want)


def test_the_output_can_be_written(fa, gpu):
    """A program that answers without no_grad, with the sinks as a parameter, and goes on in place."""
    c = make(42, "bf16", "bf16", 64, 4, 2, 16, "hnd", (40, 9), nan=False)
    t = {n: c[n].to(gpu) for n in ("q", "kp", "vp", "table", "lens", "sinks")}
    run = lambda sinks: fa.paged_attention(t["q"], t["kp"], t["vp"], t["table"], t["lens"], sinks=sinks)
    want = run(t["sinks"]) * 2 + 1
    o = run(torch.nn.Parameter(t["sinks"]))
    o.mul_(2)
    o += 1
    same(o.detach(), want)
