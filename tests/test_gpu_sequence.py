"""The sequence-block operators (layer norm, short causal convolution, selective scan) against their definitions in
float64 on the CPU (oracle/sequence_oracle.py).

Tolerance of every value: half a step of its type relative to the value (one rounding at the store; fp16 also half of its
smallest step, 2^-25, below its normal range), plus `c` fp32 roundings (2^-24) of the same sum over absolute values, which
the oracle gives.  `c` counts the roundings on the longest path to a value and is derived where it is set."""
import pytest
import torch

from oracle import sequence_oracle as SO

pytestmark = pytest.mark.gpu

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
DEV = 'cuda:0'


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _in(seed, t, *shape, scale=1.0):
    """A CPU tensor whose values are exact in type t."""
    return (_rand(seed, *shape) * scale).to(t).float()


def _gpu(v, t=torch.float32, grad=False):
    return None if v is None else v.to(DEV, t).requires_grad_(grad)


def _close(got, want, what, c):
    value, size = want
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-30
    got = got.detach().double().cpu().reshape(value.shape)
    bound = (1.01 * u * value.abs() if u > 1e-6 else 0) + c * 2.0 ** -24 * size + tiny
    off = (got - value).abs()
    if not bool((off <= bound).all()):
        i = int((off - bound).nan_to_num(float('inf')).argmax())
        raise AssertionError(f'{what}: {float(got.flatten()[i])} for {float(value.flatten()[i])}, off {float(off.flatten()[i]):.3e}, '
                             f'allowed {float(bound.flatten()[i]):.3e}; {int((off > bound).sum())} of {off.numel()}')


# ------------------------------------------------------------------ layer norm

NORM_SHAPES = [
    (1, 1, 'f32'), (1, 8, 'bf16'), (3, 2, 'f32'), (0, 16, 'f32'), (5, 300, 'f32'), (6, 301, 'bf16'), (9, 512, 'f16'),
    (700, 64, 'f32'), (4099, 24, 'bf16'), (4, 2048, 'bf16'), (3, 2056, 'f16'), (3, 1028, 'f32'), (2, 8192, 'bf16'),
    (2, 8200, 'bf16'), (3, 4100, 'f32'), (2, 16392, 'f16'), (3, 2050, 'f32'), (2, 20000, 'f32'),
]


def _norm_c(rows, H):
    # a row's sums: up to H / 64 terms in a lane, 6 to 8 joins, then a dozen single operations; the parameters' sums: the
    # rows of a workgroup in order (8 a wave at least, all rows over 512 workgroups), then the workgroups
    return H / 64 + 24, H / 64 + 24 + 8 + rows / 512 + 512 / 16 + 16


@pytest.mark.parametrize('rows,H,kind', NORM_SHAPES)
def test_layer_norm(rows, H, kind):
    from ps_vae_amd import ops
    t = TYPES[kind]
    x, w, b, dy = _in(1, t, rows, H, scale=1.5) + 0.0, 1 + 0.2 * _rand(2, H), 0.2 * _rand(3, H), _in(4, t, rows, H)
    want = SO.layer_norm(x.double(), w.double(), b.double(), 1e-5, dy.double())
    xg, wg, bg = _gpu(x, t, True), _gpu(w, grad=True), _gpu(b, grad=True)
    y = ops.layer_norm(xg, wg, bg)
    grads = torch.autograd.grad(y, (xg, wg, bg), _gpu(dy, t))
    c_row, c_par = _norm_c(rows, H)
    assert y.dtype == t and grads[0].dtype == t
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(xg, wg, bg), y)
    for got, k, c in zip((y, *grads), ('y', 'dx', 'dw', 'db'), (c_row, 2 * c_row, c_par, c_par)):
        _close(got, want[k], k, c)


def test_layer_norm_rows_far_from_zero_and_without_parameters():
    """Rows of mean 1000 and spread 1: the variance is taken about the mean, so only the inputs' own rounding shows."""
    from ps_vae_amd import ops
    x, dy = 1000 + _rand(5, 7, 333), _rand(6, 7, 333)
    for w, b in ((None, None), (1 + _rand(7, 333), None), (None, _rand(8, 333))):
        want = SO.layer_norm(x.double(), None if w is None else w.double(), None if b is None else b.double(), 1e-5, dy.double())
        xg, wg, bg = _gpu(x, grad=True), _gpu(w, grad=True), _gpu(b, grad=True)
        y = ops.layer_norm(xg, wg, bg)
        leaves = [(k, v) for k, v in (('dx', xg), ('dw', wg), ('db', bg)) if v is not None]
        grads = torch.autograd.grad(y, [v for _, v in leaves], _gpu(dy))
        _close(y, want['y'], 'y', 64)
        for (k, _), g in zip(leaves, grads):
            _close(g, want[k], k, 128)


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
def test_layer_norm_strides_and_alignment(kind):
    """Slices of wider rows, rows that begin off 16 bytes, an expanded gradient, a transposed input (copied)."""
    from ps_vae_amd import ops
    t = TYPES[kind]
    wide = _in(1, t, 6, 5, 90)
    w, b = 1 + 0.1 * _rand(2, 40), _rand(3, 40)
    g = _gpu(wide, t)
    for view, ref in ((g[..., 8:48], wide[..., 8:48]), (g[..., 1:41], wide[..., 1:41]), (g[:, 1:3, :40], wide[:, 1:3, :40]),
                      (g[..., ::2][..., :40], wide[..., ::2][..., :40]), (g[..., :40].transpose(0, 1), wide[..., :40].transpose(0, 1))):
        want = SO.layer_norm(ref.reshape(-1, 40).double(), w.double(), b.double(), 1e-5, torch.ones(ref[..., 0].numel(), 40).double())
        v = view.detach().requires_grad_()
        y = ops.layer_norm(v, _gpu(w), _gpu(b))
        _close(y, want['y'], 'y', 64)
        _close(torch.autograd.grad(y, v, torch.ones((), device=DEV, dtype=t).expand_as(y))[0], want['dx'], 'dx', 128)


def test_layer_norm_keeps_nan_and_infinity_in_their_rows():
    from ps_vae_amd import ops
    x = _rand(1, 5, 70)
    x[1, 3], x[3, 69] = float('nan'), float('inf')
    y = ops.layer_norm(_gpu(x)).cpu()
    assert bool(y[[1, 3]].isnan().any(1).all()) and bool(y[[0, 2, 4]].isfinite().all())


# ------------------------------------------------------------------ convolution

CONV_CASES = [   # (lengths, first row, rows behind, width, taps, type, state)
    ([1], 0, 0, 1, 1, 'f32', False), ([3], 0, 0, 8, 4, 'f32', True), ([0, 5, 0, 0, 1, 2, 40, 0], 2, 3, 12, 4, 'f32', True),
    ([0, 0], 0, 0, 8, 4, 'f32', True), ([0, 0], 0, 4, 8, 3, 'bf16', True), ([70, 1, 63, 64, 65], 0, 0, 600, 4, 'bf16', False),
    ([9, 30], 1, 1, 37, 2, 'f16', True), ([200, 7], 0, 0, 64, 8, 'bf16', True), ([33] * 5, 0, 0, 24, 5, 'f16', True),
    ([2, 1, 3, 1, 1, 1, 8], 0, 1, 16, 7, 'f32', True), ([500], 0, 0, 520, 6, 'f32', False), ([1] * 300, 0, 0, 40, 3, 'bf16', True),
    ([3000, 0, 1100], 5, 60, 264, 4, 'bf16', True),
]


def _packed(lengths, first, behind):
    off = SO.lengths_to_offsets(lengths, first)
    return off, off[-1] + behind, torch.tensor(off, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize('silu', [True, False])
@pytest.mark.parametrize('case', CONV_CASES, ids=lambda c: f'{len(c[0])}x{sum(c[0])}x{c[3]}-{c[4]}-{c[5]}')
def test_causal_conv(case, silu):
    from ps_vae_amd import ops
    lengths, first, behind, D, W, kind, with_state = case
    t = TYPES[kind]
    off, rows, off_gpu = _packed(lengths, first, behind)
    x, dy, w, b = _in(1, t, rows, D), _in(2, t, rows, D), _rand(3, D, W), _rand(4, D)
    state = _in(5, t, len(lengths), W - 1, D) if with_state else None
    d = lambda v: None if v is None else v.double()  # noqa: E731
    want, last = SO.causal_conv(d(x), d(w), d(b), off, d(state), silu, d(dy))
    xg, wg, bg = _gpu(x, t, True), _gpu(w, grad=True), _gpu(b, grad=True)
    y, end = ops.causal_conv(xg, wg, bg, silu=silu, seq_off=off_gpu, state=_gpu(state, t), return_state=True)
    grads = torch.autograd.grad(y, (xg, wg, bg), _gpu(dy, t))
    assert torch.equal(end.double().cpu(), last)
    # W products and a bias, the sigmoid (an exponential, a sum, a reciprocal: 6) and its products; backward twice that, the
    # W products of dx; the parameters' sums: 64 rows a lane, the stretches of a workgroup (32), the workgroups
    c = 4 * W + 16
    parts = rows / 2048 + 32 + 16
    for got, k, cc in zip((y, *grads), ('y', 'dx', 'dw', 'db'), (c, 2 * c, 2 * c + 64 + parts, 2 * c + 64 + parts)):
        _close(got, want[k], k, cc)
    with torch.no_grad():
        assert torch.equal(ops.causal_conv(xg, wg, bg, silu=silu, seq_off=off_gpu, state=_gpu(state, t)), y)


def test_causal_conv_sequences_of_one_length_are_the_packed_ones():
    from ps_vae_amd import ops
    x, w = _gpu(_rand(1, 5, 11, 20)), _gpu(_rand(2, 20, 4))
    off = torch.arange(0, 66, 11, dtype=torch.int32, device=DEV)
    y, end = ops.causal_conv(x, w, return_state=True)
    y2, end2 = ops.causal_conv(x.reshape(55, 20), w, seq_off=off, return_state=True)
    assert torch.equal(y.reshape(55, 20), y2) and torch.equal(end, end2)
    assert torch.equal(ops.causal_conv(x[2], w), y[2])


@pytest.mark.parametrize('kind,D,W', [('f32', 12, 4), ('bf16', 40, 4), ('f16', 37, 3), ('bf16', 8, 1), ('f32', 600, 8)])
def test_causal_conv_prompt_then_steps(kind, D, W):
    """A prompt in two parts and single rows give what the whole sequence gives, bit for bit (same products in the same order)."""
    from ps_vae_amd import ops
    t = TYPES[kind]
    x, w, b = _gpu(_rand(1, 3, 14, D), t), _gpu(_rand(2, D, W)), _gpu(_rand(3, D))
    whole, end = ops.causal_conv(x, w, b, silu=True, return_state=True)
    a, state = ops.causal_conv(x[:, :2], w, b, silu=True, return_state=True)
    c, state = ops.causal_conv(x[:, 2:9], w, b, silu=True, state=state, return_state=True)
    got = [a, c]
    for i in range(9, 14):
        other = torch.full_like(state, float('nan'))
        y, new = ops.causal_conv_step(x[:, i], state, w, b, silu=True, state_out=other)
        y2, same = ops.causal_conv_step(x[:, i], state, w, b, silu=True)
        assert new is other and same is state and torch.equal(y, y2) and torch.equal(other, state)
        got.append(y[:, None])
    assert torch.equal(torch.cat(got, 1), whole) and torch.equal(state, end)


@pytest.mark.parametrize('kind,D,W', [('f32', 8, 4), ('bf16', 64, 3), ('f16', 9, 8)])
def test_causal_conv_rows_behind_the_last_sequence_have_no_state(kind, D, W):
    """A stretch of rows that begins behind the last sequence, less than W - 1 rows from the end, has no state to read: what
    lies behind the states in memory reaches nothing."""
    from ps_vae_amd import ops
    t = TYPES[kind]
    states = torch.full((4, W - 1, D), float('nan'), device=DEV, dtype=t)
    states[:2] = _gpu(_rand(1, 2, W - 1, D), t)
    x, dy, w, b = _gpu(_rand(2, 66, D), t), _gpu(_rand(3, 66, D), t), _gpu(_rand(4, D, W), grad=True), _gpu(_rand(5, D), grad=True)
    off = torch.tensor([0, 3, 64], dtype=torch.int32, device=DEV)
    got = []
    for rows in (64, 65, 66):
        v = x[:rows].detach().requires_grad_()
        y = ops.causal_conv(v, w, b, silu=True, seq_off=off, state=states[:2])
        dx, dw, db = torch.autograd.grad(y, (v, w, b), dy[:rows])
        assert bool((y[64:] == 0).all()) and bool((dx[64:] == 0).all())
        got.append((y[:64], dx[:64], dw, db))
    assert all(torch.equal(p, q) and bool(p.isfinite().all()) for other in got[1:] for p, q in zip(got[0], other))


# ------------------------------------------------------------------ scan

SCAN_CASES = [   # (lengths, first row, rows behind, width, states, groups, type, flags: z D bias h0 softplus)
    ([1], 0, 0, 1, 1, 1, 'f32', 'zDbhs'), ([2], 0, 0, 5, 3, 1, 'f32', ''), ([17], 0, 0, 64, 16, 1, 'f32', 'zDbhs'),
    ([0, 5, 0, 16, 1, 33, 0, 2], 3, 2, 70, 16, 1, 'f32', 'zDbhs'), ([0, 0, 0], 0, 0, 8, 4, 1, 'f32', 'h'), ([0, 0], 0, 3, 8, 4, 2, 'bf16', 'zhs'),
    ([40, 15], 0, 0, 600, 16, 1, 'bf16', 'zDbs'), ([31, 16, 48], 1, 0, 130, 8, 2, 'f16', 'zDbhs'), ([19, 20], 0, 0, 66, 5, 1, 'bf16', 'Dh'),
    ([50, 3], 0, 0, 36, 32, 4, 'f32', 'zs'), ([23, 64], 0, 1, 40, 64, 2, 'bf16', 'zDbhs'), ([25] * 40, 0, 0, 24, 7, 3, 'f32', 'Dbs'),
    ([200], 0, 0, 12, 16, 1, 'f32', 'zDbhs'), ([90, 130], 0, 0, 37, 2, 1, 'f16', 'zDbhs'), ([64], 0, 0, 48, 33, 3, 'f32', 'zDbhs'),
]


def _scan_inputs(case):
    lengths, first, behind, width, N, G, kind, flags = case
    t = TYPES[kind]
    off, rows, off_gpu = _packed(lengths, first, behind)
    v = dict(x=_in(1, t, rows, width), dt=_in(2, t, rows, width), B=_in(3, t, rows, G, N), C=_in(4, t, rows, G, N),
             A=-(0.5 + _rand(5, width, N).abs()) * torch.arange(1, N + 1) / max(1, N // 8))
    if 's' not in flags:
        v['dt'] = v['dt'].abs() / 8
        v['dt'] = v['dt'].to(t).float()
    v['z'] = _in(6, t, rows, width) if 'z' in flags else None
    v['D'] = _rand(7, width) if 'D' in flags else None
    v['dt_bias'] = _rand(8, width).abs() / 4 - (2.0 if 's' in flags else 0.0) if 'b' in flags else None
    v['h0'] = _rand(9, len(lengths), width, N) if 'h' in flags else None
    return v, off, rows, off_gpu, 's' in flags


def _scan_c(case, v, softplus, off):
    # One row's decay: the product delta A and its scaling (2 roundings of an exponent of size m), delta's own error (8 of
    # softplus: an exponential, a logarithm, a division), the exponential's last place; the decayed term m exp(-m) bounds m
    # times it, so a row adds at most 2 + 10 / e + 4 roundings, and 3 for the update.  A gradient passes the rows twice.
    longest = max([b - a for a, b in zip(off, off[1:])] + [1])
    states = 24 + v['A'].shape[1] / 4 + 13 * longest
    sums = 2 * states + sum(b - a for a, b in zip(off, off[1:])) / 16 + 16 + 64
    return states, sums


@pytest.mark.parametrize('chunks', [-1, 1, 3])
@pytest.mark.parametrize('case', SCAN_CASES, ids=lambda c: f'{len(c[0])}x{sum(c[0])}x{c[3]}-{c[4]}-{c[5]}-{c[6]}{c[7]}')
def test_selective_scan(case, chunks):
    from ps_vae_amd import _lib, ops
    t = TYPES[case[6]]
    v, off, rows, off_gpu, softplus = _scan_inputs(case)
    dy, dhT = _in(10, t, rows, case[3]), _rand(11, len(case[0]), case[3], case[4])
    d = {k: None if q is None else q.double() for k, q in v.items()}
    want = SO.selective_scan(off=off, softplus=softplus, dy=dy.double(), dhT=dhT.double(), **d)
    leaves = {k: _gpu(q, t if k in ('x', 'dt', 'B', 'C', 'z') else torch.float32, True) for k, q in v.items()}
    old = _lib.set_option('scan_chunks', chunks)
    try:
        call = lambda: ops.selective_scan(**leaves, softplus=softplus, seq_off=off_gpu, return_state=True)  # noqa: E731
        y, last = call()
        names = [k for k, q in leaves.items() if q is not None]
        grads = dict(zip(names, torch.autograd.grad((y, last), [leaves[k] for k in names], (_gpu(dy, t), _gpu(dhT)), retain_graph=True)))
        again = torch.autograd.grad((y, last), [leaves[k] for k in names], (_gpu(dy, t), _gpu(dhT)))
        with torch.no_grad():
            y2, last2 = call()
    finally:
        _lib.set_option('scan_chunks', old)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    assert all(torch.equal(a, grads[k]) for a, k in zip(again, names))
    c, c_sum = _scan_c(case, v, softplus, off)
    _close(y, want['y'], 'y', c)
    _close(last, want['hT'], 'hT', c)
    if not rows:
        assert torch.equal(grads['h0'].cpu(), dhT) if 'h0' in grads else True
    for k, name in (('x', 'dx'), ('dt', 'ddt'), ('A', 'dA'), ('B', 'dB'), ('C', 'dC'), ('D', 'dD'), ('z', 'dz'), ('dt_bias', 'dbias'), ('h0', 'dh0')):
        if k in grads:
            _close(grads[k], want[name], name, c_sum)


@pytest.mark.parametrize('kind,width,N,G', [('f32', 12, 16, 1), ('bf16', 66, 5, 2), ('f16', 40, 64, 1), ('bf16', 256, 16, 1), ('f32', 9, 1, 3), ('f32', 30, 24, 1)])
def test_selective_scan_step(kind, width, N, G):
    """Single rows against the definition, in place and into another buffer; rows as views of wider ones."""
    from ps_vae_amd import ops
    t, S = TYPES[kind], 5
    v, off, rows, _, _ = _scan_inputs(([1] * S, 0, 0, width, N, G, kind, 'zDbhs'))
    want = SO.selective_scan(off=off, **{k: q.double() for k, q in v.items()})
    wide = torch.zeros(S, 3 * width + 3, device=DEV, dtype=t)
    views = {k: wide[:, i * (width + 1):i * (width + 1) + width] for i, k in enumerate(('x', 'dt', 'z'))}
    for k, q in views.items():
        q.copy_(v[k])
    args = {k: _gpu(v[k], t) for k in 'BC'} | {k: _gpu(v[k]) for k in ('A', 'D', 'dt_bias')} | views
    state = _gpu(v['h0'])
    other = torch.full_like(state, float('nan'))
    y, new = ops.selective_scan_step(state=state, state_out=other, **args)
    assert new is other and torch.equal(state.cpu(), v['h0'])
    y2, same = ops.selective_scan_step(state=state, **args)
    assert same is state and torch.equal(y, y2) and torch.equal(state, other)
    _close(y, want['y'], 'y', 40 + N / 4)
    _close(state, want['hT'], 'hT', 40)


def test_selective_scan_broadcast_and_shared_operands():
    """One tensor in several places, an expanded A and initial state, groupless B and C, only some gradients wanted."""
    from ps_vae_amd import ops
    L, width, N = 21, 20, 16
    x, bc, dy = _rand(1, 2, L, width), _rand(2, 2, L, N), _rand(3, 2, L, width)
    a, h = -_rand(4, N).abs(), _rand(5, N)
    off = [0, L, 2 * L]
    flat = lambda q: q.reshape(2 * L, -1).double()  # noqa: E731
    want = SO.selective_scan(flat(x), flat(x), a.expand(width, N).double(), flat(bc)[:, None], flat(bc)[:, None], off, z=flat(x),
                             h0=h.expand(2, width, N).double(), dy=flat(dy))
    xg, bg, ag, hg = (_gpu(q, grad=True) for q in (x, bc, a, h))
    y = ops.selective_scan(xg, xg, ag.expand(width, N), bg, bg, z=xg, h0=hg.expand(2, width, N))
    dx, db, da, dh = torch.autograd.grad(y, (xg, bg, ag, hg), _gpu(dy))
    c, add = 1000, lambda *k: tuple(sum(want[j][i] for j in k) for i in (0, 1))  # noqa: E731
    _close(y, want['y'], 'y', 400)
    _close(dx, add('dx', 'ddt', 'dz'), 'dx + ddt + dz', c)
    _close(db, add('dB', 'dC'), 'dB + dC', c)
    _close(da, tuple(q.sum(0) for q in want['dA']), 'dA', c)
    _close(dh, tuple(q.sum((0, 1)) for q in want['dh0']), 'dh0', c)
    # the state alone carries a gradient, too
    y, last = ops.selective_scan(xg, xg, ag.expand(width, N), bg, bg, return_state=True)
    want = SO.selective_scan(flat(x), flat(x), a.expand(width, N).double(), flat(bc)[:, None], flat(bc)[:, None], off, dy=0 * flat(dy),
                             dhT=torch.ones(2, width, N).double())
    _close(torch.autograd.grad(last.sum(), bg)[0], want['dB'], 'dB of the last state', c)


def test_scan_and_conv_leave_or_zero_rows_outside_the_sequences():
    """Through the C entry points: rows that no sequence holds stay as they were without the flag, and become zero with it."""
    import ctypes as C
    from ps_vae_amd import _lib
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    T, D, N = 12, 8, 4
    x, B = _gpu(_rand(1, T, D)), _gpu(_rand(2, T, N))
    A, w = -torch.ones(D, N, device=DEV), _gpu(_rand(3, D, 4))
    off = torch.tensor([2, 5, 9], dtype=torch.int32, device=DEV)
    outside = [0, 1, 9, 10, 11]
    sc = torch.empty(L.psvae_selective_scan_scratch_bytes(T, 2, D, 1, N, 1) + 4096, dtype=torch.uint8, device=DEV)
    kept = torch.empty(L.psvae_selective_scan_saved_bytes(T, 2, D, 1, N), dtype=torch.uint8, device=DEV)
    for flag, value in ((0, 7.0), (_lib.SEQ_ZERO_OUTSIDE, 0.0)):
        y, dx, ddt, yc, dxc = (torch.full((T, D), 7.0, device=DEV) for _ in range(5))
        dB, dC = (torch.full((T, N), 7.0, device=DEV) for _ in range(2))
        dA = torch.empty(D, N, device=DEV)
        a = _lib.Scan(x=x.data_ptr(), dt=x.data_ptr(), B=B.data_ptr(), C=B.data_ptr(), A=A.data_ptr(), ldx=D, lddt=D, ldb=N, ldc=N,
                      seq_off=off.data_ptr(), T=T, S=2, D=D, G=1, N=N, dtype=0, flags=_lib.SEQ_SOFTPLUS | flag)
        g = _lib.ScanGrads(dx=dx.data_ptr(), ddt=ddt.data_ptr(), dB=dB.data_ptr(), dC=dC.data_ptr(), dA=dA.data_ptr())
        _lib.check(L.psvae_selective_scan_forward(C.byref(a), y.data_ptr(), D, None, kept.data_ptr(), sc.data_ptr(), sc.numel(), st))
        _lib.check(L.psvae_selective_scan_backward(C.byref(a), kept.data_ptr(), x.data_ptr(), D, None, C.byref(g), sc.data_ptr(), sc.numel(), st))
        _lib.check(L.psvae_causal_conv_forward(x.data_ptr(), D, w.data_ptr(), None, yc.data_ptr(), D, off.data_ptr(), None, None, T, 2, D, 4, 0, flag, st))
        _lib.check(L.psvae_causal_conv_backward(x.data_ptr(), D, x.data_ptr(), D, w.data_ptr(), None, dxc.data_ptr(), D, None, None, off.data_ptr(), None,
                                                T, 2, D, 4, 0, flag, None, 0, st))
        for q in (y, dx, ddt, yc, dxc, dB, dC):
            assert bool((q[outside] == value).all()) and bool((q[2:9] != 7).all())


def test_offsets_that_lie_never_leave_the_rows():
    """Offsets past the rows or out of order: whatever comes out, what lies around the buffers stays as it was."""
    from ps_vae_amd import ops
    T, D, N = 40, 8, 4
    pool = torch.full((3, T, D), 3.0, device=DEV)
    x = pool[1]
    bc = _gpu(_rand(2, T, N))
    for bad in ([0, 100, 200], [50, 60, 70], [30, 10, 40], [-5, 3, 1 << 30]):
        off = torch.tensor(bad, dtype=torch.int32, device=DEV)
        xg = x.detach().requires_grad_()
        y = ops.selective_scan(ops.causal_conv(xg, torch.ones(D, 4, device=DEV), seq_off=off), xg, -torch.ones(D, N, device=DEV), bc, bc, seq_off=off)
        torch.autograd.grad(y.sum(), xg)
        torch.cuda.synchronize()
        assert bool((pool == 3).all())


def test_rows_outside_and_infinite_rates_stay_where_they_are():
    """NaN and infinity in rows that no sequence holds reach nothing; a rate of -infinity forgets its state at every row
    and nothing else, also where a sequence ends inside a tile."""
    from ps_vae_amd import ops
    off = torch.tensor([2, 13, 30], dtype=torch.int32, device=DEV)
    dirty = _rand(1, 33, 24)
    dirty[[0, 1, 30, 31, 32]] = torch.tensor([float('nan'), float('inf'), float('-inf'), float('nan'), float('inf')])[:, None]
    clean = dirty.clone()
    clean[[0, 1, 30, 31, 32]] = 0
    A = -_rand(2, 24, 8).abs()
    got = []
    for x in (dirty, clean):
        v, w, a = _gpu(x, grad=True), _gpu(_rand(3, 24, 4), grad=True), _gpu(A, grad=True)
        u = ops.causal_conv(v, w, silu=True, seq_off=off)
        y, last = ops.selective_scan(u, v, a, v[:, :8], v[:, 8:16], z=v, seq_off=off, return_state=True)
        got.append([y, last, *torch.autograd.grad((y, last), (v, w, a), (_gpu(_rand(4, 33, 24)), torch.ones_like(last)))])
    assert all(torch.equal(p, q) and bool(p.isfinite().all()) for p, q in zip(*got))
    A[:, 3], x = float('-inf'), _gpu(clean[2:30])
    y, last = ops.selective_scan(x, x, _gpu(A), x[:, :8], x[:, 8:16], h0=torch.ones(1, 24, 8, device=DEV), return_state=True)
    step = torch.nn.functional.softplus(x[-1]) * x[-1]
    assert bool(y.isfinite().all()) and torch.allclose(last[0, :, 3], step * x[-1, 3], rtol=1e-5, atol=1e-6)


def test_more_elements_than_32_bits_count():
    """2.2 G elements an operand: the last rows and sequences come out as they do by themselves, bit for bit."""
    from ps_vae_amd import ops
    S, L, D, few = 135_000, 16, 1024, 3
    tail = [_gpu(_rand(i, few, L, D), torch.bfloat16) for i in range(2)]
    x, dt = (torch.zeros(S, L, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    x[-few:], dt[-few:] = tail
    w, A = _gpu(_rand(3, D, 4)), -_gpu(_rand(4, D, 1).abs())
    ones = torch.ones(1, device=DEV, dtype=torch.bfloat16)

    def run(x, dt):
        x, dt = x.requires_grad_(), dt.requires_grad_()
        bc = ones.expand(*x.shape[:2], 1)
        n = ops.layer_norm(x)
        u = ops.causal_conv(n, w, silu=True)
        y, last = ops.selective_scan(u, dt, A, bc, bc, return_state=True)
        dx, ddt = torch.autograd.grad(y, (x, dt), ones.expand_as(y))
        return [q[-few:].clone() for q in (n, u, y, last, dx, ddt)]
    alone = run(tail[0].clone(), tail[1].clone())
    whole = run(x, dt)
    assert x.numel() > 2 ** 31 and all(torch.equal(a, b) for a, b in zip(alone, whole))
    state = torch.zeros(S, D, 16, device=DEV)                       # 2.2 G states, 8.8 GB
    state[-few:] = 1
    row = torch.ones(S, D, device=DEV, dtype=torch.bfloat16)
    bc = torch.ones(S, 16, device=DEV, dtype=torch.bfloat16)
    rates = A.expand(D, 16).contiguous()
    y, _ = ops.selective_scan_step(row, row, rates, bc, bc, state)
    ya, sa = ops.selective_scan_step(row[:few], row[:few], rates, bc[:few], bc[:few], torch.ones(few, D, 16, device=DEV))
    assert torch.equal(y[-few:], ya) and torch.equal(state[-few:], sa)


def test_more_work_than_one_launch_takes():
    """Rows and sequences beyond 2^23 workgroups go into further launches or turns: the last ones come out as they do by
    themselves, bit for bit."""
    from ps_vae_amd import ops
    few, bf16 = 5, torch.bfloat16

    def zeros(rows, *shape):
        v = torch.zeros(rows, *shape, device=DEV, dtype=bf16)
        v[-few:] = _gpu(_rand(1, few, *shape), bf16)
        return v

    def alike(f, x):
        for whole, alone in zip(f(x), f(x[-few:].clone())):
            assert bool(alone.isfinite().all()) and torch.equal(whole[-few:], alone)

    def norm(x):
        x = x.detach().requires_grad_()
        y = ops.layer_norm(x)
        return y.detach(), torch.autograd.grad(y, x, x.detach())[0]
    for rows, width in ((1 << 25, 8), (1 << 23, 257), (1 << 23, 1025)):   # a wave, a workgroup a row; backward in two readings
        alike(norm, zeros(rows + few + 3, width))
    D = 1025
    w = _gpu(_rand(2, D, 8))
    alike(lambda x: ops.causal_conv_step(x, torch.empty(len(x), 0, D, device=DEV, dtype=bf16), w[:, :1].contiguous())[:1], zeros((1 << 21) + few, D))
    alike(lambda x: ops.causal_conv(x, w[:160], return_state=True), zeros((1 << 21) + few, 1, 160))
    A = -_gpu(_rand(3, 1024, 1).abs())

    def step(x):
        state = torch.ones(len(x), 1024, 1, device=DEV)
        return ops.selective_scan_step(x, x, A, x[:, :1], x[:, 1:2], state, z=x)
    alike(step, zeros((1 << 19) + few, 1024))


# ------------------------------------------------------------------ refusals

def test_operators_refuse_what_they_do_not_take():
    from ps_vae_amd import ops
    x, w = torch.zeros(6, 8, device=DEV), torch.zeros(8, 4, device=DEV)
    off = torch.tensor([0, 6], dtype=torch.int32, device=DEV)
    A, bc = torch.zeros(8, 4, device=DEV), torch.zeros(6, 4, device=DEV)
    norm, conv, scan = ops.layer_norm, ops.causal_conv, ops.selective_scan
    state = torch.zeros(6, 8, 4, device=DEV)
    for f in (
        lambda: norm(x.double()), lambda: norm(x.int()), lambda: norm(x, torch.ones(7, device=DEV)), lambda: norm(x, torch.ones(8)),
        lambda: norm(torch.zeros((), device=DEV)), lambda: norm(torch.zeros(3, 0, device=DEV)),
        lambda: conv(x, torch.zeros(8, 9, device=DEV)), lambda: conv(x, w[:7]), lambda: conv(x[None], w, seq_off=off), lambda: conv(x, w, seq_off=off.long()),
        lambda: conv(x, w, seq_off=off.cpu()), lambda: conv(x, w, seq_off=off[:1]), lambda: conv(x, w, state=torch.zeros(1, 2, 8, device=DEV)),
        lambda: conv(x, w, state=torch.zeros(1, 3, 8, device=DEV, requires_grad=True)), lambda: conv(x, w, state=torch.zeros(1, 3, 8, device=DEV).half()),
        lambda: ops.causal_conv_step(x, torch.zeros(6, 3, 8, device=DEV).transpose(0, 1).contiguous().transpose(0, 1), w),
        lambda: scan(x, x.half(), A, bc, bc), lambda: scan(x, x, A[:7], bc, bc), lambda: scan(x, x, A, bc[:5], bc), lambda: scan(x, x, A, bc, bc[:, :3]),
        lambda: scan(x, x, torch.zeros(8, 65, device=DEV), bc, bc), lambda: scan(x, x, A, bc[:, None].expand(6, 3, 4), bc[:, None].expand(6, 3, 4)),
        lambda: scan(x, x, A, bc, bc, z=x[:5]), lambda: scan(x, x, A, bc, bc, h0=torch.zeros(2, 8, 4, device=DEV)), lambda: scan(x, x, A.int(), bc, bc),
        lambda: ops.selective_scan_step(x, x, A, bc, bc, state.half()), lambda: ops.selective_scan_step(x, x, A, bc, bc, state[:5]),
        lambda: ops.selective_scan_step(x, x, A, bc, bc, torch.zeros(7, 8, 4, device=DEV)[:6], state_out=state[:5]),
    ):
        with pytest.raises(ValueError):
            f()
    both = torch.zeros(7, 8, 4, device=DEV)
    with pytest.raises(ValueError, match='overlaps'):
        ops.selective_scan_step(x, x, A, bc, bc, both[:6], state_out=both[1:])
    with pytest.raises(RuntimeError, match='no backward'):
        ops.selective_scan_step(x.clone().requires_grad_(), x, A, bc, bc, state)
    # gradients are not differentiable again: asking for a graph of them is fine, using it is refused
    v = torch.ones(6, 8, device=DEV, requires_grad=True)
    for y in (norm(v), conv(v, w + 1), scan(v, v, A - 1, bc + 1, bc + 1)):
        g, = torch.autograd.grad((y * y).sum(), v, create_graph=True)
        with pytest.raises(RuntimeError, match='once_differentiable'):
            g.sum().backward()


# ------------------------------------------------------------------ the operators together

def _block_reference(m, x, off, h0):
    """SSMBlock.forward in float64 on the CPU, through the oracle's definitions and torch products."""
    p = {k: q.detach().double().cpu() for k, q in m.state_dict().items()}
    n, _ = SO.layer_norm(x, p['norm.weight'], p['norm.bias'], 1e-5)['y']
    u, z = (n @ p['in_proj.weight'].t()).chunk(2, -1)
    (v, _), = SO.causal_conv(u, p['conv_weight'], p['conv_bias'], off)[0].values()
    r = v @ p['x_proj.weight'].t()
    gn = m.num_groups * m.num_states
    B, C = (r[:, m.dt_rank + i * gn:m.dt_rank + (i + 1) * gn].reshape(-1, m.num_groups, m.num_states) for i in range(2))
    out = SO.selective_scan(v, r[:, :m.dt_rank] @ p['dt_proj.weight'].t(), -torch.exp(p['A_log']), B, C, off, p['D'], z, p['dt_proj.bias'], h0=h0)
    return x + out['y'][0] @ p['out_proj.weight'].t(), out['hT'][0]


def _block(dim=24, **kw):
    from ps_vae_amd import SSMBlock
    torch.manual_seed(3)
    return SSMBlock(dim, **kw).to(DEV)


def test_block_forward_prompt_and_steps():
    """Ragged prompts against the definitions; a prompt followed by single rows gives what the whole sequences give."""
    m = _block(num_groups=2)
    x = _rand(1, 3, 20, 24)
    off = [0, 20, 40, 60]
    want, hT = _block_reference(m, x.reshape(60, 24).double(), off, None)
    with torch.no_grad():
        whole, (window, h) = m(_gpu(x), return_state=True)
        # five layers of sums of up to 48 terms of size one, relative to values of size one: 1e-5 is 170 roundings
        assert torch.allclose(whole.double().cpu().reshape(60, 24), want, rtol=1e-5, atol=1e-5)
        assert torch.allclose(h.double().cpu(), hT, rtol=1e-5, atol=1e-5)
        packed = m(_gpu(x).reshape(60, 24), seq_off=torch.tensor(off, dtype=torch.int32, device=DEV))
        assert torch.allclose(packed.reshape(3, 20, 24), whole, rtol=1e-5, atol=1e-5)
        part, state = m(_gpu(x)[:, :13], return_state=True)
        rows = [part] + [m.step(_gpu(x)[:, i], state)[:, None] for i in range(13, 20)]
        assert torch.allclose(torch.cat(rows, 1), whole, rtol=1e-5, atol=1e-5)
        assert torch.allclose(state[0], window, rtol=1e-5, atol=1e-5) and torch.allclose(state[1], h, rtol=1e-5, atol=1e-5)
        fresh = m.init_state(3)
        rows = [m.step(_gpu(x)[:, i], fresh)[:, None] for i in range(20)]
        assert torch.allclose(torch.cat(rows, 1), whole, rtol=1e-5, atol=1e-5)


def test_block_gradients_against_differences():
    """Every parameter's gradient along a random direction against a central difference of the float64 definitions.  The
    difference is off by h^2 times a third derivative, the fp32 gradient by a few hundred roundings of its terms."""
    m = _block()
    x, weight = _rand(1, 31, 24), _rand(2, 31, 24)
    off = [0, 11, 11, 31]
    off_gpu = torch.tensor(off, dtype=torch.int32, device=DEV)
    loss = (m(_gpu(x), seq_off=off_gpu) * _gpu(weight)).sum()
    names, params = zip(*m.named_parameters())
    grads = torch.autograd.grad(loss, params)
    for i, (name, p, g) in enumerate(zip(names, params, grads)):
        v = _rand(50 + i, *p.shape).double()
        v /= v.norm()
        with torch.no_grad():
            keep, ends = p.detach().clone(), []
            m.double()
            for sign in (1, -1):
                p.copy_(keep.double() + sign * 1e-4 * v.to(DEV))
                ends.append(float((_block_reference(m, x.double(), off, None)[0] * weight.double()).sum()))
            m.float()
            p.copy_(keep)
        slope = (ends[0] - ends[1]) / 2e-4
        got = float((g.double().cpu() * v).sum())
        assert abs(got - slope) <= 1e-4 * (float((g.double().cpu() * v).abs().sum()) + 1e-3), (name, got, slope)


def test_block_on_another_stream_and_in_a_graph():
    """The block on a side stream, and its forward and backward captured into one graph: every replay, with eager work of
    the same parameters between, gives the eager bits; two graphs have workspaces of their own."""
    m = _block()
    off = torch.tensor([0, 7, 40, 64], dtype=torch.int32, device=DEV)
    params = list(m.parameters())
    xs = [_gpu(_rand(s, 64, 24)) for s in (1, 2)]

    def work(x):
        y = m(x, seq_off=off)
        return [y.detach(), *torch.autograd.grad(y, params, torch.ones_like(y))]
    want = [work(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = work(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs, ins = [], [], [x.clone() for x in xs]
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(work(x))
        graphs.append(g)
    for turn in range(4):
        order = (0, 1) if turn % 2 else (1, 0)
        for i in order:
            ins[i].copy_(xs[(i + turn) % 2])
            graphs[i].replay()
        eager = work(xs[turn % 2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[turn % 2]))
        for i in order:
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[(i + turn) % 2])), (turn, i)


def test_block_captured_while_an_eager_graph_of_it_lives():
    """A capture of forward and backward over aliases of the parameters (p.detach().requires_grad_()), while an eager graph
    of the parameters themselves is alive: aliases have gradient nodes of their own, on the capturing stream."""
    m = _block()
    x = _gpu(_rand(1, 2, 30, 24))
    params = dict(m.named_parameters())
    alive = m(x)
    want = torch.autograd.grad(alive, list(params.values()), torch.ones_like(alive), retain_graph=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        alias = {k: p.detach().requires_grad_() for k, p in params.items()}
        y = torch.func.functional_call(m, alias, (x,))
        got = torch.autograd.grad(y, list(alias.values()), torch.ones_like(y))
    for _ in range(3):
        g.replay()
        again = torch.autograd.grad(alive, list(params.values()), torch.ones_like(alive), retain_graph=True)
        torch.cuda.synchronize()
        assert torch.equal(y, alive) and all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, want, again))


def test_steps_in_a_graph():
    """A decoding step captured once and replayed moves its state on as eager steps do."""
    m = _block()
    x = _gpu(_rand(1, 6, 4, 24))
    eager = m.init_state(4)
    want = [m.step(x[i], eager) for i in range(6)]
    state, row = m.init_state(4), x[0].clone()
    m.step(row, m.init_state(4))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m.step(row, state)
    for q in state:
        q.zero_()
    for i in range(6):
        row.copy_(x[i])
        g.replay()
        assert torch.equal(y, want[i])
    assert all(torch.equal(a, b) for a, b in zip(state, eager))


def test_steps_in_place_are_seen_by_a_backward_pass_that_kept_the_state():
    """A state that a convolution's backward pass reads and a token step has moved on since is refused, not used; in
    inference mode, where nothing is kept, steps go on."""
    from ps_vae_amd import ops
    x, w = _gpu(_rand(1, 2, 5, 8), grad=True), _gpu(_rand(2, 8, 4))
    A, bc = -torch.ones(8, 4, device=DEV), torch.ones(2, 4, device=DEV)
    for into in (False, True):
        state = torch.ones(2, 3, 8, device=DEV)
        y = ops.causal_conv(x, w, state=state)
        ops.causal_conv_step(x[:, 0].detach(), state.clone() if into else state, w, state_out=state if into else None)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.sum().backward()
    h = torch.ones(2, 8, 4, device=DEV)
    kept = (h * h.clone().requires_grad_()).sum()
    ops.selective_scan_step(x[:, 0].detach(), x[:, 1].detach(), A, bc, bc, h)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        kept.backward()
    with torch.inference_mode():
        state = torch.ones(2, 3, 8, device=DEV)
        before = state.clone()
        ops.causal_conv_step(x[:, 0].detach(), state, w)
        assert not torch.equal(state, before)


@pytest.mark.parametrize('shape', [(0, 5, 8), (2, 0, 8), (0, 8)])
def test_no_rows_give_no_rows_and_zero_gradients(shape):
    """No sequences, or only empty ones; the block's Linear kernels refuse what has no rows, before a state is touched."""
    from ps_vae_amd import ops
    off = torch.zeros(1, dtype=torch.int32, device=DEV) if len(shape) == 2 else None
    S = shape[0]
    x, w, A = torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(8, 4, device=DEV, requires_grad=True), -torch.ones(8, 2, device=DEV)
    A.requires_grad_()
    h0, bc = torch.ones(S, 8, 2, device=DEV, requires_grad=True), torch.zeros(*shape[:-1], 2, device=DEV)
    gain = torch.ones(8, device=DEV, requires_grad=True)
    u, end = ops.causal_conv(ops.layer_norm(x, gain, gain), w, seq_off=off, state=torch.ones(S, 3, 8, device=DEV), return_state=True)
    y, last = ops.selective_scan(u, u, A, bc, bc, D=gain, h0=h0, seq_off=off, return_state=True)
    assert y.shape == shape and bool((end == 1).all()) and end.shape == (S, 3, 8) and torch.equal(last, h0)
    grads = torch.autograd.grad(y.sum() + last.sum(), (x, w, A, gain, h0))
    assert [g.shape for g in grads] == [v.shape for v in (x, w, A, gain, h0)]
    assert all(bool((g == 0).all()) for g in grads[:4]) and bool((grads[4] == 1).all())
    rows = torch.zeros(0, 8, device=DEV)
    with torch.no_grad():
        ops.causal_conv_step(rows, torch.ones(0, 3, 8, device=DEV), w)
        ops.selective_scan_step(rows, rows, A, rows[:, :2], rows[:, :2], torch.ones(0, 8, 2, device=DEV))
        m, state = _block(8), torch.ones(shape[0], 3, 16, device=DEV)
        with pytest.raises(RuntimeError):
            m(x, seq_off=off, state=(state, torch.ones(shape[0], 16, 16, device=DEV)))
        assert bool((state == 1).all())


def test_block_trained_in_segments_cuts_the_gradient_at_their_border():
    """Two segments with a detached state between them: the loss of the whole sequence, each parameter's gradient the sum of
    the two segments' own.  A state that is not detached is refused, in the next call and in the backward pass."""
    m, x = _block(), _gpu(_rand(1, 3, 20, 24))
    params = list(m.parameters())
    first, state = m(x[:, :9], return_state=True)
    with pytest.raises(ValueError, match='detached'):
        m(x[:, 9:], state=state)
    with pytest.raises(RuntimeError, match='no gradient is computed for the state'):
        torch.autograd.grad(state[0].sum(), params[0], retain_graph=True)
    state = [s.detach() for s in state]
    second = m(x[:, 9:], state=state)
    with torch.no_grad():
        assert torch.allclose(torch.cat([first, second], 1), m(x), rtol=1e-5, atol=1e-5)
    together = torch.autograd.grad(first.sum() + second.sum(), params, retain_graph=True)
    apart = [torch.autograd.grad(y.sum(), params) for y in (first, second)]
    # the engine adds the same two terms, in fp32
    assert all(torch.equal(t, a + b) for t, a, b in zip(together, *apart))


def _scan_with(dt, A, chunks, **kw):
    """(outputs by name, oracle's outputs) of a scan of 96 rows of one sequence, in `chunks` pieces; no softplus."""
    from ps_vae_amd import _lib, ops
    v = {k: q for k, q in kw.items() if k not in ('dy', 'dhT')} | dict(dt=dt, A=A)
    d = {k: q.double() for k, q in kw.items()} | dict(dt=dt.double(), A=A.double())
    want = SO.selective_scan(off=[0, 96], softplus=False, **d)
    leaves = {k: _gpu(q, grad=True) for k, q in v.items()}
    old = _lib.set_option('scan_chunks', chunks)
    try:
        y, last = ops.selective_scan(**leaves, softplus=False, return_state=True)
        grads = torch.autograd.grad((y, last), list(leaves.values()), (_gpu(kw['dy']), _gpu(kw['dhT'])))
    finally:
        _lib.set_option('scan_chunks', old)
    names = dict(x='dx', dt='ddt', A='dA', B='dB', C='dC', h0='dh0')
    return {'y': y, 'hT': last, **{names[k]: g for k, g in zip(leaves, grads)}}, want


# The pieces of 96 rows are 32 rows each.  A piece's decay as a whole is exp of a sum of 32 steps, whose argument of size m
# is off by m 2^-24 a step's rounding; rows one by one have the same.  13 roundings a row as for every scan above, and as
# many again for larger arguments (three rows of 30, three roundings each; 3.5 elsewhere), once for the state and twice for a
# gradient.
_PIECES_C, _PIECES_C_GRAD = 2 * 13 * 96 + 32, 4 * 13 * 96 + 64


@pytest.mark.parametrize('chunks', [1, 3])
def test_growing_pieces_leave_a_state_of_zero_alone(chunks):
    """Positive rates: a piece grows what enters it by more than fp32 holds (2^140 and more), but what enters is zero.  The
    rows give finite values one by one, and so do the pieces, forward (no inputs before the second piece) and backward (no
    gradients behind it)."""
    rows, width, N = 96, 8, 4
    A = 0.9 + 0.1 * torch.rand(width, N, generator=torch.Generator().manual_seed(1))
    dt = torch.full((rows, width), 0.125)
    dt[:32] = dt[64:] = 3.5                               # 32 x 3.5 x 0.9 = 101 and more: 145 bits
    dt[32:35] = dt[61:64] = -30.0                         # what the middle passes on has lost 81 and more
    middle = torch.zeros(rows, 1)
    middle[35:61] = 1
    args = dict(x=_rand(2, rows, width) * middle, dy=_rand(3, rows, width) * middle, B=_rand(4, rows, 1, N), C=_rand(5, rows, 1, N),
                dhT=torch.zeros(1, width, N))
    bits = (dt[:32].double()[..., None] * A.double()).sum(0) / 0.6931471805599453
    assert float(bits.min()) > 128
    got, want = _scan_with(dt, A, chunks, **args)
    for k in got:
        assert bool(got[k].isfinite().all()), k
        _close(got[k], want[k], k, _PIECES_C if k in ('y', 'hT') else _PIECES_C_GRAD)


@pytest.mark.parametrize('chunks', [1, 3])
def test_fading_pieces_keep_what_is_left_of_a_large_state(chunks):
    """A piece's decay below 2^-126 does not become zero in front of a state of 2^100: what is left of it is an ordinary
    number.  The same backward with a large gradient of the last state."""
    rows, width, N = 96, 8, 4
    A = -(0.9 + 0.1 * torch.rand(width, N, generator=torch.Generator().manual_seed(1)))
    zero, big = torch.zeros(rows, width), _rand(2, 1, width, N) * 2.0 ** 100
    bc = dict(B=_rand(3, rows, 1, N), C=_rand(4, rows, 1, N))
    dt = torch.full((rows, width), 0.125)
    dt[:32] = 3.25                                        # 32 x 3.25 x 0.9 = 93 and more: 135 bits
    got, want = _scan_with(dt, A, chunks, x=zero, dy=zero, h0=big, dhT=torch.zeros(1, width, N), **bc)
    assert float(want['y'][0][32:].abs().min()) > 1e-20
    for k in ('y', 'hT'):
        _close(got[k], want[k], k, _PIECES_C)
    got, want = _scan_with(dt.flip(0), A, chunks, x=zero, dy=zero, h0=torch.zeros(1, width, N), dhT=big, **bc)
    assert float(want['dx'][0][:64].abs().min()) > 1e-20
    for k in ('dx', 'dh0'):
        _close(got[k], want[k], k, _PIECES_C_GRAD)


class _Fenced:
    """Tensors in the middle of larger ones: inputs between NaN, outputs between sevens that have to stay."""

    def __init__(self, t):
        self.t, self.outs = t, []

    def _place(self, shape, value, dtype):
        n = 1
        for s in shape:
            n *= s
        pool = torch.full((n + 2 * 4096,), value, device=DEV, dtype=dtype)
        return pool, pool[4096:4096 + n].view(shape)

    def input(self, v, dtype=None):
        pool, mid = self._place(v.shape, float('nan'), dtype or self.t)
        mid.copy_(v)
        return mid

    def output(self, *shape, dtype=None):
        pool, mid = self._place(shape, 7.0, dtype or self.t)
        self.outs.append((pool, mid))
        return mid

    def check(self, what):
        torch.cuda.synchronize()
        for i, (pool, mid) in enumerate(self.outs):
            assert bool((pool[:4096] == 7).all()) and bool((pool[4096 + mid.numel():] == 7).all()), (what, i, 'fence')
            assert bool(mid.isfinite().all()), (what, i, 'a row from outside came in')


@pytest.mark.parametrize('flag', [0, 4])
@pytest.mark.parametrize('kind,D,N,W', [('f32', 8, 4, 4), ('bf16', 37, 5, 8), ('f16', 64, 33, 3)])
@pytest.mark.parametrize('bad', [[0, 100, 200], [50, 60, 70], [30, 10, 40], [-5, 3, 1 << 30], [2 ** 31 - 1, -2 ** 31, 20], [39, 40, 39]], ids=str)
def test_no_access_leaves_the_rows_whatever_the_offsets_hold(bad, kind, D, N, W, flag):
    """Convolution and scan, forward, backward and states, in one piece and in three: nothing around any output changes, and
    nothing around any input (NaN there) reaches a value.  What the values are is left open."""
    import ctypes as C
    from ps_vae_amd import _lib
    L, st, t, f32 = _lib.lib(), torch.cuda.current_stream().cuda_stream, TYPES[kind], torch.float32
    T, S, G, code = 40, 2, 1, {'f32': 0, 'bf16': 1, 'f16': 2}[kind]
    assert flag in (0, _lib.SEQ_ZERO_OUTSIDE)
    for chunks in (1, 3):
        f = _Fenced(t)
        x, dt, z, dy = (f.input(_rand(i, T, D)) for i in range(4))
        B, Cm = (f.input(_rand(4 + i, T, G * N)) for i in range(2))
        A, h0, dhT = f.input(-_rand(6, D, N).abs(), f32), f.input(_rand(7, S, D, N), f32), f.input(_rand(8, S, D, N), f32)
        w, vec, state = f.input(_rand(9, D, W), f32), f.input(_rand(10, D), f32), f.input(_rand(11, S, W - 1, D))
        off = torch.tensor([-7] + bad + [1 << 30], dtype=torch.int32, device=DEV)[1:4]
        y, dx, ddt, dz, yc, dxc = (f.output(T, D) for _ in range(6))
        dB, dC = f.output(T, G * N), f.output(T, G * N)
        dA, dD, dbias, hT, dh0 = f.output(D, N, dtype=f32), f.output(D, dtype=f32), f.output(D, dtype=f32), f.output(S, D, N, dtype=f32), f.output(S, D, N, dtype=f32)
        dw, db, state_out = f.output(D, W, dtype=f32), f.output(D, dtype=f32), f.output(S, W - 1, D)
        old = _lib.set_option('scan_chunks', chunks)
        try:
            sizes = [L.psvae_selective_scan_saved_bytes(T, S, D, G, N), L.psvae_selective_scan_scratch_bytes(T, S, D, G, N, 0),
                     L.psvae_selective_scan_scratch_bytes(T, S, D, G, N, 1), L.psvae_causal_conv_scratch_bytes(T, D, W, code)]
            assert all(n % 4 == 0 for n in sizes) and (sizes[1] > 0) == (chunks > 1)
            kept, fwd, bwd, conv = (f.output(n // 4, dtype=f32) for n in sizes)
            a = _lib.Scan(x=x.data_ptr(), dt=dt.data_ptr(), B=B.data_ptr(), C=Cm.data_ptr(), z=z.data_ptr(), ldx=D, lddt=D, ldb=G * N, ldc=G * N, ldz=D,
                          A=A.data_ptr(), skip=vec.data_ptr(), dt_bias=vec.data_ptr(), h0=h0.data_ptr(), seq_off=off.data_ptr(), T=T, S=S, D=D, G=G, N=N,
                          dtype=code, flags=_lib.SEQ_SOFTPLUS | flag)
            g = _lib.ScanGrads(dx=dx.data_ptr(), ddt=ddt.data_ptr(), dB=dB.data_ptr(), dC=dC.data_ptr(), dz=dz.data_ptr(), dA=dA.data_ptr(),
                               d_skip=dD.data_ptr(), d_dt_bias=dbias.data_ptr(), dh0=dh0.data_ptr())
            _lib.check(L.psvae_selective_scan_forward(C.byref(a), y.data_ptr(), D, hT.data_ptr(), kept.data_ptr(), fwd.data_ptr(), sizes[1], st))
            _lib.check(L.psvae_selective_scan_backward(C.byref(a), kept.data_ptr(), dy.data_ptr(), D, dhT.data_ptr(), C.byref(g), bwd.data_ptr(), sizes[2], st))
        finally:
            _lib.set_option('scan_chunks', old)
        _lib.check(L.psvae_causal_conv_forward(x.data_ptr(), D, w.data_ptr(), vec.data_ptr(), yc.data_ptr(), D, off.data_ptr(), state.data_ptr(),
                                               state_out.data_ptr(), T, S, D, W, code, _lib.SEQ_SILU | flag, st))
        _lib.check(L.psvae_causal_conv_backward(dy.data_ptr(), D, x.data_ptr(), D, w.data_ptr(), vec.data_ptr(), dxc.data_ptr(), D, dw.data_ptr(), db.data_ptr(),
                                                off.data_ptr(), state.data_ptr(), T, S, D, W, code, _lib.SEQ_SILU | flag, conv.data_ptr(), sizes[3], st))
        f.check((chunks, flag))
