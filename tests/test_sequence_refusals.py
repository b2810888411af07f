"""What the sequence-block operators refuse before they reach the library.  The library call is stubbed, so no GPU is
needed: a call that gets as far as the stub was not refused."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from ps_vae_amd import ops


class Launched(Exception):
    pass


@pytest.fixture(autouse=True)
def _stub(monkeypatch):
    def run(*args):
        raise Launched
    monkeypatch.setattr(ops, '_need_gpu', lambda t, what: None)
    monkeypatch.setattr(ops, '_run', run)


def _operands():
    """{entry point: (call, its tensors by name)} over sizes that every check accepts."""
    x, rows, states = torch.ones(6, 8), torch.ones(6, 4), torch.ones(6, 8, 4)
    w, A, v = torch.ones(8, 4), -torch.ones(8, 4), torch.ones(8)
    return {
        'layer_norm': (ops.layer_norm, dict(x=x, weight=v, bias=v)),
        'causal_conv': (ops.causal_conv, dict(x=x, weight=w, bias=v, state=torch.ones(1, 3, 8))),
        'causal_conv_step': (ops.causal_conv_step, dict(x=x, state=torch.ones(6, 3, 8), weight=w, bias=v, state_out=torch.ones(6, 3, 8))),
        'selective_scan': (ops.selective_scan, dict(x=x, dt=x, A=A, B=rows, C=rows, D=v, z=x, dt_bias=v, h0=states[:1])),
        'selective_scan_step': (ops.selective_scan_step, dict(x=x, dt=x, A=A, B=rows, C=rows, state=states, D=v, z=x, dt_bias=v,
                                                              state_out=states.clone())),
    }


@pytest.mark.parametrize('name', list(_operands()))
def test_operands_with_a_tangent_are_refused(name):
    """Forward-mode differentiation: a result without a tangent would stand for a derivative of zero."""
    call, args = _operands()[name]
    with fwd.dual_level():
        with pytest.raises(Launched):                     # an open level alone changes nothing
            call(**args)
        for k, v in args.items():
            dual = {**args, k: fwd.make_dual(v, torch.ones_like(v))}
            for mode in (torch.enable_grad, torch.no_grad):   # neither switches forward mode off
                with mode(), pytest.raises(RuntimeError, match='forward-mode'):
                    call(**dual)
            with torch.inference_mode(), pytest.raises(Launched):   # this does, for every operator of torch
                call(**dual)
    with pytest.raises(Launched):
        call(**args)
