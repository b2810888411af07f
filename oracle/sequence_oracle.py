"""Layer norm, the short causal convolution and the selective scan from their definitions, in float64 on the CPU, with
their gradients written out.  Test infrastructure only.

Every function also returns what the same sums come to over absolute values: an fp32 evaluation of a sum is off by at
most a small multiple of 2^-24 times that, whatever cancels in it, so the tests' tolerances are made from it."""
import torch


def lengths_to_offsets(lengths, first=0):
    off = [first]
    for n in lengths:
        off.append(off[-1] + n)
    return off


def layer_norm(x, w, b, eps, dy=None):
    """{name: (value, magnitude)} of y and, given dy, of dx, dw, db.  The magnitudes hold the error of the row's mean and
    of xhat: both are sums over the row."""
    H = x.shape[-1]
    w = torch.ones(H, dtype=x.dtype) if w is None else w
    b = torch.zeros(H, dtype=x.dtype) if b is None else b
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    xhat = (x - mean) * rstd
    size = x.abs().mean(-1, keepdim=True)
    # xhat's own error: of x - mean, relative to |x| and the mean's terms, and of rstd, relative to xhat
    mx = rstd * (x.abs() + size) + xhat.abs()
    out = {'y': (xhat * w + b, mx * w.abs() + b.abs())}
    if dy is None:
        return out
    g = dy * w
    s0, s1 = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
    m0, m1 = g.abs().mean(-1, keepdim=True), (g.abs() * (mx + xhat.abs())).mean(-1, keepdim=True)
    out['dx'] = (rstd * (g - s0 - xhat * s1), rstd * (g.abs() + m0 + xhat.abs() * m1 + mx * s1.abs()))
    out['dw'] = ((dy * xhat).sum(0), (dy.abs() * mx).sum(0))
    out['db'] = (dy.sum(0), dy.abs().sum(0))
    return out


def _silu(v):
    s = torch.sigmoid(v)
    return v * s, s * (1 + v * (1 - s))


def causal_conv(x, w, b, off, state=None, silu=True, dy=None):
    """Rows outside the sequences give zeros.  Returns ({name: (value, magnitude)}, final state)."""
    rows, D = x.shape
    W = w.shape[1]
    b = torch.zeros(D, dtype=x.dtype) if b is None else b
    S = len(off) - 1
    state = torch.zeros(S, W - 1, D, dtype=x.dtype) if state is None else state
    y, my, dx, mdx = (torch.zeros_like(x) for _ in range(4))
    dw, mdw, db, mdb = torch.zeros_like(w), torch.zeros_like(w), torch.zeros_like(b), torch.zeros_like(b)
    last = torch.zeros_like(state)
    for s in range(S):
        o, e = off[s], off[s + 1]
        n = e - o
        full = torch.cat([state[s], x[o:e]])
        last[s] = full[full.shape[0] - (W - 1):]
        if n == 0:
            continue
        win = torch.stack([full[k:k + n] for k in range(W)])                       # [W, n, D]
        pre = (win * w.t()[:, None]).sum(0) + b
        mag = (win * w.t()[:, None]).abs().sum(0) + b.abs()
        act, slope = _silu(pre) if silu else (pre, torch.ones_like(pre))
        y[o:e], my[o:e] = act, mag                                                 # |silu'| < 1.1
        if dy is None:
            continue
        g = dy[o:e] * slope
        mg = dy[o:e].abs() * (1 + mag) if silu else dy[o:e].abs()                  # |silu''| < 1/2
        for k in range(W):
            back = W - 1 - k
            m = n - back
            if m > 0:
                dx[o:o + m] += w[:, k] * g[back:]
                mdx[o:o + m] += w[:, k].abs() * mg[back:]
        dw += (win * g).sum(1).t()
        mdw += (win.abs() * mg).sum(1).t()
        db += g.sum(0)
        mdb += mg.sum(0)
    out = {'y': (y, my)}
    if dy is not None:
        out.update(dx=(dx, mdx), dw=(dw, mdw), db=(db, mdb))
    return out, last


def _scan_core(a, delta, A, x, B, C, D, h0, dyp=None, dhT=None):
    """One sequence: a, [L, width, N]; delta, x, dyp [L, width]; B, C [L, width, N].  Linear in every operand, so that the
    same code over absolute values gives the magnitudes."""
    L = x.shape[0]
    h, hs = h0, []
    for t in range(L):
        h = a[t] * h + (delta[t] * x[t])[:, None] * B[t]
        hs.append(h)
    hs = torch.stack(hs) if L else a
    y = (hs * C).sum(-1) + D * x
    if dyp is None:
        return y, h, None
    before = torch.cat([h0[None], hs[:-1]]) if L else hs
    carry = dhT
    g = torch.zeros_like(a)
    for t in reversed(range(L)):
        g[t] = C[t] * dyp[t][:, None] + carry
        carry = a[t] * g[t]
    by_b = (g * B).sum(-1)
    dec = g * a * before
    return y, h, dict(dx=by_b * delta + D * dyp, ddelta=by_b * x + (dec * A).sum(-1), dA=(dec * delta[..., None]).sum(0),
                      dB=g * (delta * x)[..., None], dC=hs * dyp[..., None], dD=(dyp * x).sum(0), dh0=carry)


def selective_scan(x, dt, A, B, C, off, D=None, z=None, dt_bias=None, softplus=True, h0=None, dy=None, dhT=None):
    """B, C [rows, G, N].  Returns {name: (value, magnitude)} with y, hT and, given dy, every gradient."""
    (rows, width), N, G, S = x.shape, A.shape[1], B.shape[1], len(off) - 1
    zero = torch.zeros(width, dtype=x.dtype)
    D_ = zero if D is None else D
    v = dt + (zero if dt_bias is None else dt_bias)
    delta = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v
    slope = torch.sigmoid(v) if softplus else torch.ones_like(v)
    gate, dgate = _silu(z) if z is not None else (torch.ones_like(x), None)
    spread = lambda q: q.repeat_interleave(width // G, 1)  # noqa: E731
    h0_ = torch.zeros(S, width, N, dtype=x.dtype) if h0 is None else h0
    dhT_ = torch.zeros_like(h0_) if dhT is None else dhT
    names = ['y', 'hT'] + (['dx', 'ddt', 'dA', 'dB', 'dC', 'dD', 'dz', 'dbias', 'dh0'] if dy is not None else [])
    shape = dict(y=x, hT=h0_, dx=x, ddt=x, dA=A, dB=B, dC=C, dD=zero, dz=x, dbias=zero, dh0=h0_)
    out = {k: (torch.zeros_like(shape[k]), torch.zeros_like(shape[k])) for k in names}
    group = lambda q: q.reshape(q.shape[0], G, width // G, N).sum(2)  # noqa: E731
    for s in range(S):
        r = slice(off[s], off[s + 1])
        a = torch.exp(delta[r][..., None] * A)
        dyp = None if dy is None else dy[r] * gate[r]
        for i, f in enumerate((lambda q: q, torch.abs)):
            y, h, g = _scan_core(a, f(delta[r]), f(A), f(x[r]), f(spread(B[r])), f(spread(C[r])), f(D_), f(h0_[s]),
                                 None if dy is None else f(dyp), f(dhT_[s]))
            out['y'][i][r] = y * f(gate[r])
            out['hT'][i][s] = h
            if dy is None:
                continue
            out['dx'][i][r] = g['dx']
            out['ddt'][i][r] = g['ddelta'] * slope[r]
            out['dA'][i].add_(g['dA'])
            out['dB'][i][r] = group(g['dB'])
            out['dC'][i][r] = group(g['dC'])
            out['dD'][i].add_(g['dD'])
            out['dbias'][i].add_((g['ddelta'] * slope[r]).sum(0))
            out['dh0'][i][s] = g['dh0']
            if z is not None:
                out['dz'][i][r] = f(dy[r]) * y * f(dgate[r])
    return out
