"""The float64 definitions that the sequence-block kernels are held to (oracle/sequence_oracle.py) against torch's
autograd and against central differences, and the operators' refusals that need no GPU."""
import ctypes as C

import pytest
import torch

from oracle import sequence_oracle as SO

F64 = torch.float64


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


def _difference(f, args, i, direction, h=1e-5):
    up, down = list(args), list(args)
    up[i], down[i] = args[i] + h * direction, args[i] - h * direction
    return (f(*up) - f(*down)) / (2 * h)


def _check(f, args, grads):
    """f(*args) -> scalar; grads[i] against autograd and against a central difference along a random direction.
    The difference is off by h^2 / 6 times a third derivative (1e-11 here) and by rounding, 1e-16 / h = 1e-11, times the
    loss's own size."""
    leaves = [a.clone().requires_grad_() for a in args]
    auto = torch.autograd.grad(f(*leaves), leaves)
    for i, (g, want) in enumerate(zip(grads, auto)):
        assert torch.allclose(g, want, rtol=1e-10, atol=1e-11), i
        v = _rand(99 + i, *args[i].shape)
        slope = float((g * v).sum())
        size = float(f(*args).abs()) + float((g * v).abs().sum()) + 1
        assert abs(float(_difference(f, args, i, v)) - slope) < 1e-7 * size, i


def test_layer_norm():
    x, w, b, dy = _rand(1, 5, 7), _rand(2, 7), _rand(3, 7), _rand(4, 5, 7)
    out = SO.layer_norm(x, w, b, 1e-5, dy)
    assert torch.allclose(out['y'][0], torch.nn.functional.layer_norm(x, (7,), w, b, 1e-5), rtol=1e-12)
    _check(lambda x, w, b: (SO.layer_norm(x, w, b, 1e-5)['y'][0] * dy).sum(), (x, w, b), [out[k][0] for k in ('dx', 'dw', 'db')])


@pytest.mark.parametrize('silu', [True, False])
@pytest.mark.parametrize('W', [1, 2, 4])
def test_causal_conv(W, silu):
    off = [1, 4, 4, 5, 11]                      # a row outside, an empty sequence, one shorter than the filter
    x, w, b, dy, state = _rand(1, 12, 3), _rand(2, 3, W), _rand(3, 3), _rand(4, 12, 3), _rand(5, 4, W - 1, 3)
    out, last = SO.causal_conv(x, w, b, off, state, silu, dy)
    assert torch.equal(last[1], state[1]) and (W == 1 or torch.equal(last[3][-1], x[10]))
    _check(lambda x, w, b: (SO.causal_conv(x, w, b, off, state, silu)[0]['y'][0] * dy).sum(), (x, w, b),
           [out[k][0] for k in ('dx', 'dw', 'db')])


@pytest.mark.parametrize('softplus,gate', [(True, True), (False, False)])
def test_selective_scan(softplus, gate):
    off, width, N, G = [0, 3, 3, 8], 4, 3, 2
    x, dt, B, Cm, z = _rand(1, 9, width), _rand(2, 9, width).abs(), _rand(3, 9, G, N), _rand(4, 9, G, N), _rand(5, 9, width)
    A, D, bias, h0 = -_rand(6, width, N).abs(), _rand(7, width), _rand(8, width).abs(), _rand(9, 3, width, N)
    dy, dhT = _rand(10, 9, width), _rand(11, 3, width, N)

    def loss(x, dt, A, B, Cm, D, z, bias, h0):
        o = SO.selective_scan(x, dt, A, B, Cm, off, D, z if gate else None, bias, softplus, h0)
        return (o['y'][0] * dy).sum() + (o['hT'][0] * dhT).sum()
    args = (x, dt, A, B, Cm, D, z, bias, h0)
    out = SO.selective_scan(x, dt, A, B, Cm, off, D, z if gate else None, bias, softplus, h0, dy, dhT)
    keys = ['dx', 'ddt', 'dA', 'dB', 'dC', 'dD', 'dz', 'dbias', 'dh0']
    if not gate:
        args, keys = args[:6] + args[7:], keys[:6] + keys[7:]
        f = lambda *a: loss(*a[:6], None, *a[6:])  # noqa: E731
    else:
        f = loss
    _check(f, args, [out[k][0] for k in keys])
    assert all(bool((out[k][1] >= out[k][0].abs() - 1e-12).all()) for k in keys)


def test_c_entry_points_refuse_bad_arguments():
    """Argument errors come back as codes before anything is launched (no GPU is touched)."""
    from ps_vae_amd import _lib
    L = _lib.lib()
    E_NULL, E_SHAPE, E_ALIGN, E_WORKSPACE = -1, -2, -3, -4
    p = 4096                                   # an address that is never followed
    assert L.psvae_layer_norm_forward(p, 7, None, None, p, 8, None, None, 2, 8, 1e-5, 0, None) == E_SHAPE      # ldx < width
    assert L.psvae_layer_norm_forward(p, 8, None, None, p, 8, None, None, 2, 8, 1e-5, 3, None) == E_SHAPE      # unknown type
    assert L.psvae_layer_norm_forward(None, 8, None, None, p, 8, None, None, 2, 8, 1e-5, 0, None) == E_NULL
    assert L.psvae_layer_norm_forward(None, 8, None, None, None, 8, None, None, 0, 8, 1e-5, 0, None) == 0      # no rows
    assert L.psvae_layer_norm_scratch_bytes(-1, 8) == 0 and L.psvae_layer_norm_scratch_bytes(5, 8) >= 64
    n = L.psvae_layer_norm_scratch_bytes(5, 8)
    bwd = lambda scratch, nbytes: L.psvae_layer_norm_backward(p, 8, p, 8, None, p, p, p, 8, p, p, 5, 8, 0, scratch, nbytes, None)  # noqa: E731
    assert bwd(None, n) == E_NULL and bwd(p + 4, n) == E_ALIGN and bwd(p, n - 1) == E_WORKSPACE

    conv = lambda W=4, T=6, S=2, flags=1, ldx=8, out=None, off=None: L.psvae_causal_conv_forward(  # noqa: E731
        p, ldx, p, None, p, 8, off, None, out, T, S, 8, W, 0, flags, None)
    assert conv(W=0) == E_SHAPE and conv(W=9) == E_SHAPE and conv(T=7) == E_SHAPE and conv(ldx=4) == E_SHAPE and conv(flags=2) == E_SHAPE
    assert conv(S=0, T=3, off=p) == E_SHAPE
    assert L.psvae_causal_conv_forward(p, 8, None, None, p, 8, None, None, None, 6, 2, 8, 4, 0, 0, None) == E_NULL
    assert L.psvae_causal_conv_forward(p, 8, p, None, p, 8, None, p, p, 6, 2, 8, 4, 0, 0, None) == E_SHAPE     # state_out is state
    assert L.psvae_causal_conv_step(p, 8, None, None, p, None, p, 8, 2, 8, 4, 0, 0, None) == E_NULL
    n = L.psvae_causal_conv_scratch_bytes(6, 8, 4, 0)
    assert L.psvae_causal_conv_backward(p, 8, p, 8, p, None, p, 8, p, p, None, None, 6, 2, 8, 4, 0, 1, p, n - 1, None) == E_WORKSPACE

    def scan(**over):
        f = dict(x=p, dt=p, B=p, C=p, A=p, ldx=8, lddt=8, ldb=4, ldc=4, T=6, S=2, D=8, G=1, N=4, dtype=0, flags=2)
        return _lib.Scan(**{**f, **over})
    fwd = lambda **over: L.psvae_selective_scan_forward(scan(**over), p, 8, None, None, None, 0, None)  # noqa: E731
    for bad in (dict(T=7), dict(N=0), dict(N=65, ldb=65, ldc=65), dict(G=3), dict(G=0), dict(D=0), dict(ldx=7), dict(ldb=3), dict(dtype=9), dict(flags=1),
                dict(S=-1), dict(z=p, ldz=0)):
        assert fwd(**bad) == E_SHAPE, bad
    for bad in (dict(x=None), dict(A=None), dict(C=None)):
        assert fwd(**bad) == E_NULL, bad
    assert L.psvae_selective_scan_forward(None, p, 8, None, None, None, 0, None) == E_NULL
    assert L.psvae_selective_scan_step(scan(T=6, S=2), p, 8, p, None) == E_SHAPE                               # T != S
    assert L.psvae_selective_scan_step(scan(T=2, S=2), p, 8, p, None) == E_NULL                                # no h0
    g = _lib.ScanGrads(dx=p, ddt=p, dB=p, dC=p, dA=p)
    n = L.psvae_selective_scan_scratch_bytes(6, 2, 8, 1, 4, 1)
    back = lambda scratch, nbytes, saved=p: L.psvae_selective_scan_backward(scan(), saved, p, 8, None, g, scratch, nbytes, None)  # noqa: E731
    assert back(p, n - 1) == E_WORKSPACE and back(p + 4, n) == E_ALIGN and back(p, n, None) == E_NULL and back(None, n) == E_NULL
    old = _lib.set_option('scan_chunks', 3)
    try:                                                                                                      # a cut time axis needs scratch
        assert L.psvae_selective_scan_scratch_bytes(600, 1, 8, 1, 4, 0) > 0
        assert fwd() == E_NULL
        assert L.psvae_selective_scan_forward(scan(), p, 8, None, None, p, 16, None) == E_WORKSPACE
    finally:
        _lib.set_option('scan_chunks', old)
    assert C.sizeof(_lib.Scan) == 8 * 15 + 8 + 24 and C.sizeof(_lib.ScanGrads) == 8 * 9


def test_operators_refuse_cpu_tensors():
    from ps_vae_amd import modules, ops
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match='GPU'):
        ops.layer_norm(x)
    with pytest.raises(RuntimeError, match='GPU'):
        ops.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match='GPU'):
        ops.selective_scan(x, x, torch.zeros(8, 4), x[:, :4], x[:, :4])
    with pytest.raises(RuntimeError, match='GPU'):
        modules.SSMBlock(8)(x)
    for bad in (dict(num_states=65), dict(num_taps=9), dict(num_groups=3)):
        with pytest.raises(ValueError):
            modules.SSMBlock(8, **bad)
