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


def _returned_state(monkeypatch, x, w):
    monkeypatch.setattr(ops, '_run', lambda *args: None)
    return ops.causal_conv(x, w, return_state=True)


def test_the_convolutions_state_passes_no_gradient_on_unnoticed(monkeypatch):
    """The state that a call returns depends on its rows.  No gradient is computed for a state, so one that has not been
    detached is refused by the next call, and a gradient of it by the backward pass, instead of being left out."""
    x, w = torch.ones(6, 8, requires_grad=True), torch.ones(8, 4, requires_grad=True)
    y, state = _returned_state(monkeypatch, x, w)
    assert state.requires_grad
    with pytest.raises(ValueError, match='detach'):
        ops.causal_conv(x, w, state=state)
    with pytest.raises(RuntimeError, match='no gradient is computed for the state'):
        torch.autograd.grad(y.sum() + state.sum(), x)
    ops.causal_conv(x, w, state=state.detach())
    with torch.no_grad():                                 # nothing is left out where no gradient is wanted
        ops.causal_conv(x, w, state=state)


@pytest.mark.parametrize('x_grad,taps', [(False, 4), (True, 1)])
def test_a_state_that_depends_on_no_leaf_needs_no_detaching(monkeypatch, x_grad, taps):
    """Rows that are data, or one tap, whose state is empty."""
    x, w = torch.ones(6, 8, requires_grad=x_grad), torch.ones(8, taps, requires_grad=True)
    y, state = _returned_state(monkeypatch, x, w)
    assert y.requires_grad and not state.requires_grad
    ops.causal_conv(x, w, state=state)


def test_block_refuses_a_state_of_its_own_that_is_not_detached(monkeypatch):
    """Training in segments: with the window's share missing, the gradient would be neither the whole one nor the one that
    is cut at the segments' border."""
    from ps_vae_amd import modules
    monkeypatch.setattr(ops, '_run', lambda *args: None)
    monkeypatch.setattr(ops, 'linear', torch.nn.functional.linear)
    m, x = modules.SSMBlock(8), torch.ones(2, 5, 8)
    y, state = m(x, return_state=True)
    with pytest.raises(ValueError, match='detached'):
        m(x, state=state)
    m(x, state=[s.detach() for s in state])
    m(x, state=(state[0].detach(), state[1]))             # the scan's state by itself carries its whole gradient
    with torch.no_grad():
        m(x, state=state)


@pytest.mark.parametrize('spoil', [lambda h: h[:3], lambda h: h.half(), lambda h: h[..., :3].contiguous(), lambda h: h.transpose(0, 1).contiguous().transpose(0, 1)],
                         ids=['sequences', 'type', 'states', 'order'])
def test_block_step_moves_both_parts_of_a_state_or_neither(monkeypatch, spoil):
    """A scan state that is refused is refused before the convolution's part has been moved on in place."""
    from ps_vae_amd import modules
    calls = []
    monkeypatch.setattr(ops, '_run', lambda what, *args: calls.append(what))
    monkeypatch.setattr(ops, 'linear', torch.nn.functional.linear)
    m = modules.SSMBlock(8, num_states=4)
    window, h = m.init_state(5)
    with pytest.raises(ValueError, match='state'):
        m.step(torch.ones(5, 8), (window, spoil(h)))
    assert 'psvae_causal_conv_step' not in calls
    m.step(torch.ones(5, 8), (window, h))
    assert calls[-2:] == ['psvae_causal_conv_step', 'psvae_selective_scan_step']


@pytest.mark.parametrize('name', ['causal_conv_step', 'selective_scan_step'])
def test_token_steps_refuse_every_operand_that_requires_a_gradient(name):
    """`state_out` too: it would go on requiring a gradient, with values that have no history."""
    call, args = _operands()[name]
    for k, v in args.items():
        wants = {**args, k: v.clone().requires_grad_()}
        with pytest.raises(RuntimeError, match='no backward pass'):
            call(**wants)
        with torch.no_grad(), pytest.raises(Launched):
            call(**wants)
