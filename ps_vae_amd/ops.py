"""Single-operator autograd functions over the C ABI (the module-level API uses
these; the whole-step path in `model.py` bypasses them)."""
import torch
from torch.autograd import forward_ad

from . import _lib


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _need_gpu(t, what):
    if not t.is_cuda:
        raise RuntimeError(f'{what}: tensors must live on the GPU; ps_vae_amd has no CPU implementation')


def _f32c(t):
    return t.contiguous().float()


def _scratch(nbytes, device):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


class LinearFn(torch.autograd.Function):
    """y = act(x w^T + b) over the last dimension (nn.Linear semantics)."""

    @staticmethod
    def forward(ctx, x, w, b, relu):
        _need_gpu(x, 'linear')
        L = _lib.lib()
        shape = x.shape
        x2 = _f32c(x).reshape(-1, shape[-1])
        w, bb = _f32c(w), (None if b is None else _f32c(b))
        M, K, N = x2.shape[0], x2.shape[1], w.shape[0]
        y = torch.empty(M, N, dtype=torch.float32, device=x.device)
        sc = _scratch(L.psvae_linear_scratch_bytes(M, N, K, 1), x.device)
        _lib.check(L.psvae_linear_forward(x2.data_ptr(), K, w.data_ptr(), None if bb is None else bb.data_ptr(),
                                          y.data_ptr(), N, M, N, K, int(relu), sc.data_ptr(), sc.numel(), _stream()),
                   'psvae_linear_forward')
        ctx.save_for_backward(x2, w, y if relu else None)
        ctx.has_bias, ctx.relu, ctx.shape = b is not None, bool(relu), shape
        return y.reshape(*shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        L = _lib.lib()
        x2, w, y = ctx.saved_tensors
        M, K, N = x2.shape[0], x2.shape[1], w.shape[0]
        dy2 = _f32c(dy).reshape(M, N)
        if ctx.relu:
            dy2 = dy2 * (y > 0)   # gradient gate of the fused ReLU
        dx = torch.empty(M, K, dtype=torch.float32, device=dy.device)
        _lib.check(L.psvae_linear_backward_input(dy2.data_ptr(), N, w.data_ptr(), dx.data_ptr(), K, M, N, K, None, 0, 0,
                                                 _stream()), 'psvae_linear_backward_input')
        dw = torch.empty_like(w)
        db = torch.empty(N, dtype=torch.float32, device=dy.device) if ctx.has_bias else None
        sc = _scratch(L.psvae_linear_scratch_bytes(M, N, K, 1), dy.device)
        _lib.check(L.psvae_linear_backward_weight(dy2.data_ptr(), N, 0, x2.data_ptr(), K, 0, 1, dw.data_ptr(),
                                                  None if db is None else db.data_ptr(), M, N, K, sc.data_ptr(), sc.numel(),
                                                  _stream()), 'psvae_linear_backward_weight')
        return dx.reshape(ctx.shape), dw, db, None


def linear(x, w, b=None, relu=False):
    return LinearFn.apply(x, w, b, relu)


class Csr:
    """By-target and by-source CSR of an edge list, built with index ops on the
    tensors' own device (stable sorts keep the edge order inside every row)."""

    def __init__(self, edge_index, edge_type, n):
        src, dst = edge_index[0].long(), edge_index[1].long()
        self.n, self.E = int(n), int(src.numel())
        dev = src.device

        def build(rows, cols):
            order = torch.sort(rows, stable=True).indices
            ptr = torch.zeros(n + 1, dtype=torch.int32, device=dev)
            if rows.numel():
                ptr[1:] = torch.cumsum(torch.bincount(rows, minlength=n), 0).to(torch.int32)
            return ptr, cols[order].to(torch.int32).contiguous(), edge_type[order].to(torch.int32).contiguous()
        self.rowptr, self.col, self.etype = build(dst, src)
        self.rowptr_t, self.col_t, self.etype_t = build(src, dst)


class GineAggregateFn(torch.autograd.Function):
    """out_i = (1+eps) x_i + sum_{j->i} relu(x_j + edge_w[:, type] + edge_b)."""

    @staticmethod
    def forward(ctx, x, edge_w, edge_b, csr, one_plus_eps):
        _need_gpu(x, 'gine_aggregate')
        L = _lib.lib()
        x, edge_w, edge_b = _f32c(x), _f32c(edge_w), _f32c(edge_b)
        n, H = x.shape
        out = torch.empty_like(x)
        _lib.check(L.psvae_gine_aggregate_forward(x.data_ptr(), H, csr.rowptr.data_ptr(), csr.col.data_ptr(),
                                                  csr.etype.data_ptr(), edge_w.data_ptr(), edge_b.data_ptr(),
                                                  float(one_plus_eps), out.data_ptr(), H, n, H, _stream()),
                   'psvae_gine_aggregate_forward')
        ctx.save_for_backward(x, edge_w, edge_b)
        ctx.csr, ctx.ope = csr, float(one_plus_eps)
        return out

    @staticmethod
    def backward(ctx, da):
        L = _lib.lib()
        x, edge_w, edge_b = ctx.saved_tensors
        csr, n, H = ctx.csr, x.shape[0], x.shape[1]
        da = _f32c(da)
        dx = torch.empty_like(x)
        dw, db = torch.zeros_like(edge_w), torch.zeros_like(edge_b)
        part = torch.empty(max(1, L.psvae_gine_edge_grad_scratch(n, H)), dtype=torch.float32, device=x.device)
        _lib.check(L.psvae_gine_aggregate_backward(da.data_ptr(), H, x.data_ptr(), H, csr.rowptr_t.data_ptr(),
                                                   csr.col_t.data_ptr(), csr.etype_t.data_ptr(), edge_w.data_ptr(),
                                                   edge_b.data_ptr(), ctx.ope, None, 0, None, dx.data_ptr(), H,
                                                   dw.data_ptr(), db.data_ptr(), part.data_ptr(), n, H, _stream()),
                   'psvae_gine_aggregate_backward')
        return dx, dw, db, None, None


class SegmentPoolFn(torch.autograd.Function):
    """pooled[b] = sum of the rows graph_off[b] .. graph_off[b+1] (rows grouped by graph)."""

    @staticmethod
    def forward(ctx, x, graph_off, node_graph):
        _need_gpu(x, 'segment_pool')
        L = _lib.lib()
        x = _f32c(x)
        n, W = x.shape
        B = graph_off.numel() - 1
        pooled = torch.empty(B, W, dtype=torch.float32, device=x.device)
        _lib.check(L.psvae_segment_pool_forward(x.data_ptr(), W, graph_off.data_ptr(), pooled.data_ptr(), W, B, W, _stream()),
                   'psvae_segment_pool_forward')
        ctx.save_for_backward(node_graph)
        ctx.n = n
        return pooled

    @staticmethod
    def backward(ctx, dp):
        L = _lib.lib()
        (node_graph,) = ctx.saved_tensors
        dp = _f32c(dp)
        W = dp.shape[1]
        dx = torch.empty(ctx.n, W, dtype=torch.float32, device=dp.device)
        _lib.check(L.psvae_gine_aggregate_backward(None, 0, None, 0, None, None, None, None, None, 1.0, dp.data_ptr(), W,
                                                   node_graph.data_ptr(), dx.data_ptr(), W, None, None, None, ctx.n, W,
                                                   _stream()),
                   'psvae_gine_aggregate_backward(pool broadcast)')
        return dx, None, None


# ---- sequence-block operators: layer norm, short causal convolution, selective scan -----------------------------
# Activations are fp32, bf16 or fp16 (one type a call), [.., width]; rows may be strided views (a slice of a wider
# projection) and are copied only where their last dimension is not contiguous.  Parameters and states are fp32.
# Sequences are either the first dimension of a [S, L, width] tensor or, with `seq_off` (int32 [S+1] on the same device,
# non-decreasing), rows seq_off[s] .. seq_off[s+1]-1 of a packed [T, width] tensor; without it [T, width] is one
# sequence.  Packed rows that no sequence holds give zeros and get zero gradients.

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _run(what, device, fn, *args):
    """The library call on the device's current stream, with that device current."""
    index = device.index
    if index == torch.cuda.current_device():
        # the handle alone: the Stream object of torch.cuda.current_stream() costs 2.7 us, as much as a launch
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, what)


def _once(backward):
    """A backward that cannot be differentiated again; the guard that says so is gone through only where somebody may."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _ptr(t):
    return None if t is None else t.data_ptr()


def _written(t):
    """Tells autograd that the library wrote into `t`, so that a backward pass that kept it says so instead of using it."""
    if not t.is_inference():                               # those have no version to count
        torch.autograd.graph.increment_version(t)


def _rows(t, width):
    """`t` as rows of `width` contiguous elements and the distance of two rows; a copy only where no view does it."""
    if t.is_contiguous():
        return t, width
    t = t.reshape(-1, width)
    if (width > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < width):
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else width)


def _act(what, name, t, like, shape):
    """Checks an activation operand against the call's first one."""
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f'{what}: {name} is {t.dtype} on {t.device}, x is {like.dtype} on {like.device}')
    if t.shape != shape:
        raise ValueError(f'{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}')


def _par(what, name, t, like, shape):
    """A parameter or state: checked, fp32, contiguous."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f'{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}')
    if t.device != like.device:
        raise ValueError(f'{what}: {name} is on {t.device}, x is on {like.device}')
    if t.dtype is torch.float32:
        return t if t.is_contiguous() else t.contiguous()
    if not t.is_floating_point():
        raise ValueError(f'{what}: {name} is {t.dtype}, expected a floating type')
    return t.float().contiguous()


def _first(what, x, low, high):
    _need_gpu(x, what)
    if x.dtype not in _DTYPES:
        raise ValueError(f'{what}: x is {x.dtype}; float32, bfloat16 and float16 are supported')
    if not low <= x.dim() <= high:
        raise ValueError(f'{what}: x has {x.dim()} dimensions')
    if x.shape[-1] < 1:
        raise ValueError(f'{what}: x has no channels')


def _sequences(what, x, seq_off):
    """(rows, sequences) of x."""
    rows = x.shape[0] if x.dim() == 2 else x.shape[0] * x.shape[1]
    if seq_off is None:
        return rows, (1 if x.dim() == 2 else x.shape[0])
    if x.dim() != 2:
        raise ValueError(f'{what}: seq_off goes with packed rows [T, width], x has {x.dim()} dimensions')
    if seq_off.dtype is not torch.int32 or seq_off.dim() != 1 or not seq_off.is_contiguous() or seq_off.device != x.device or not len(seq_off):
        raise ValueError(f'{what}: seq_off must be a contiguous int32 vector of sequences + 1 offsets on {x.device}')
    if seq_off.numel() == 1 and rows:
        raise ValueError(f'{what}: seq_off names no sequence for {rows} rows')
    return rows, seq_off.numel() - 1


def _no_tangent(what, *tensors):
    """Refuses operands of forward-mode differentiation: the kernels read the values alone, and a result without a tangent
    would stand for a derivative of zero."""
    # no level is open almost always; unpacking nine operands to find that out would cost as much as a launch
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f'{what} has no forward-mode derivative: its operands must not carry tangents')


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _norm_forward(x, w, b, eps, keep):
    H, dev = x.shape[-1], x.device
    rows = x.numel() // H
    x2, ldx = _rows(x, H)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    stats, mean, rstd = None, None, None
    if keep:
        stats = torch.empty(2, rows, dtype=torch.float32, device=dev)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    _run('psvae_layer_norm_forward', dev, _lib.lib().psvae_layer_norm_forward, x2.data_ptr(), ldx, _ptr(w), _ptr(b), y.data_ptr(), H, mean, rstd,
         rows, H, eps, _DTYPES[x.dtype])
    return y, x2, ldx, stats


class LayerNormFn(torch.autograd.Function):
    """y = (x - mean) / sqrt(var + eps) * w + b over the last dimension."""

    @staticmethod
    def forward(ctx, x, w, b, eps):
        y, x2, ctx.ldx, stats = _norm_forward(x, w, b, eps, True)
        ctx.save_for_backward(x2, w, stats)
        ctx.shape = x.shape
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        L = _lib.lib()
        x2, w, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad      # False where the operand was None
        shape, rows, dev, dtype = ctx.shape, stats.shape[1], stats.device, x2.dtype
        H = shape[-1]
        dy2, lddy = _rows(dy, H)
        dx = torch.empty(shape, dtype=dtype, device=dev) if need_x else None
        dw = torch.empty(H, dtype=torch.float32, device=dev) if need_w else None
        db = torch.empty(H, dtype=torch.float32, device=dev) if need_b else None
        nbytes = L.psvae_layer_norm_scratch_bytes(rows, H) if need_w or need_b else 0
        sc = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        mean = stats.data_ptr()
        _run('psvae_layer_norm_backward', dev, L.psvae_layer_norm_backward, dy2.data_ptr(), lddy, x2.data_ptr(), ctx.ldx, _ptr(w), mean,
             mean + 4 * rows, _ptr(dx), H, _ptr(dw), _ptr(db), rows, H, _DTYPES[dtype], _ptr(sc), nbytes)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension of x [.., H]; weight and bias [H], each optional."""
    _first('layer_norm', x, 1, 64)
    shape = x.shape[-1:]
    weight, bias = _par('layer_norm', 'weight', weight, x, shape), _par('layer_norm', 'bias', bias, x, shape)
    _no_tangent('layer_norm', x, weight, bias)
    if _wants_grad(x, weight, bias):
        return LayerNormFn.apply(x, weight, bias, float(eps))
    return _norm_forward(x, weight, bias, float(eps), False)[0]


def _conv_forward(x, w, b, state, seq_off, flags, rows, S, want_state):
    (D, W), dev = w.shape, x.device
    x2, ldx = _rows(x, D)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    out = torch.empty(S, W - 1, D, dtype=x.dtype, device=dev) if want_state else None
    _run('psvae_causal_conv_forward', dev, _lib.lib().psvae_causal_conv_forward, x2.data_ptr(), ldx, w.data_ptr(), _ptr(b), y.data_ptr(), D,
         _ptr(seq_off), _ptr(state), _ptr(out), rows, S, D, W, _DTYPES[x.dtype], flags)
    return y, out, x2, ldx


class CausalConvFn(torch.autograd.Function):
    """y[t] = act(b + sum_k w[:, k] x[t - W + 1 + k]) inside every sequence; returns (y, final state or None).  The state has
    no gradient: backward refuses one."""

    @staticmethod
    def forward(ctx, x, w, b, state, seq_off, flags, rows, S, want_state):
        y, out, x2, ldx = _conv_forward(x, w, b, state, seq_off, flags, rows, S, want_state)
        ctx.save_for_backward(x2, w, b, state, seq_off)
        ctx.call = ldx, flags, rows, S, x.shape
        ctx.set_materialize_grads(False)
        # the state holds rows of x: it requires a gradient as they do, so that one that is passed on is noticed
        if out is not None and not (out.shape[1] and ctx.needs_input_grad[0]):
            ctx.mark_non_differentiable(out)
        return y, out

    @staticmethod
    @_once
    def backward(ctx, dy, dout):
        if dout is not None:
            raise RuntimeError('causal_conv: no gradient is computed for the state; detach it')
        L = _lib.lib()
        x2, w, b, state, seq_off = ctx.saved_tensors
        ldx, flags, rows, S, shape = ctx.call
        need_x, need_w, need_b = ctx.needs_input_grad[:3]     # False where the operand was None
        (D, W), dev, dtype = w.shape, w.device, x2.dtype
        dy2, lddy = _rows(dy, D)
        dx = torch.empty(shape, dtype=dtype, device=dev) if need_x else None
        dw = torch.empty(D, W, dtype=torch.float32, device=dev) if need_w else None
        db = torch.empty(D, dtype=torch.float32, device=dev) if need_b else None
        code = _DTYPES[dtype]
        nbytes = L.psvae_causal_conv_scratch_bytes(rows, D, W, code) if need_w or need_b else 0
        sc = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        _run('psvae_causal_conv_backward', dev, L.psvae_causal_conv_backward, dy2.data_ptr(), lddy, x2.data_ptr(), ldx, w.data_ptr(), _ptr(b),
             _ptr(dx), D, _ptr(dw), _ptr(db), _ptr(seq_off), _ptr(state), rows, S, D, W, code, flags, _ptr(sc), nbytes)
        return dx, dw, db, None, None, None, None, None, None


def _conv_params(what, x, weight, bias):
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= 8:
        raise ValueError(f'{what}: weight has shape {tuple(weight.shape)}, expected [channels, taps] with 1 to 8 taps')
    D = x.shape[-1]
    return _par(what, 'weight', weight, x, (D, weight.shape[1])), _par(what, 'bias', bias, x, (D,))


def causal_conv(x, weight, bias=None, *, silu=False, seq_off=None, state=None, return_state=False):
    """Short causal convolution along every sequence, one filter a channel: weight [D, W] with 1 to 8 taps (the last one
    on the row itself), bias [D].  `state` [S, W-1, D] in x's type holds the inputs in front of every sequence (oldest
    first; zeros without it); with `return_state` the call gives (y, state behind the end).  No gradient is computed for a
    state: where one would be needed the call refuses, so the returned state is passed on as state.detach()."""
    what = 'causal_conv'
    _first(what, x, 2, 3)
    rows, S = _sequences(what, x, seq_off)
    weight, bias = _conv_params(what, x, weight, bias)
    if state is not None:
        _act(what, 'state', state, x, (S, weight.shape[1] - 1, x.shape[-1]))
        if _wants_grad(state):
            raise ValueError(f'{what}: no gradient is computed for the state; pass state.detach()')
        state = state.contiguous()
    _no_tangent(what, x, weight, bias, state)
    flags = (_lib.SEQ_SILU if silu else 0) | (_lib.SEQ_ZERO_OUTSIDE if seq_off is not None else 0)
    if _wants_grad(x, weight, bias):
        y, out = CausalConvFn.apply(x, weight, bias, state, seq_off, flags, rows, S, bool(return_state))
    else:
        y, out = _conv_forward(x, weight, bias, state, seq_off, flags, rows, S, return_state)[:2]
    return (y, out) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, silu=False, state_out=None):
    """One row x [S, D] for each of S sequences.  `state` [S, W-1, D] is moved on by the row, in place or into
    `state_out`; returns (y, the new state).  No gradients."""
    what = 'causal_conv_step'
    _first(what, x, 2, 2)
    S, D = x.shape
    weight, bias = _conv_params(what, x, weight, bias)
    _no_tangent(what, x, state, weight, bias, state_out)
    if _wants_grad(x, state, weight, bias, state_out):
        raise RuntimeError(f'{what} has no backward pass: call it under torch.no_grad() or on detached tensors')
    _act(what, 'state', state, x, (S, weight.shape[1] - 1, D))
    out = _state_out(what, state, state_out)
    x2, ldx = _rows(x, D)
    y = torch.empty(S, D, dtype=x.dtype, device=x.device)
    _run('psvae_causal_conv_step', x.device, _lib.lib().psvae_causal_conv_step, x2.data_ptr(), ldx, state.data_ptr(), out.data_ptr(), weight.data_ptr(),
         _ptr(bias), y.data_ptr(), D, S, D, weight.shape[1], _DTYPES[x.dtype], _lib.SEQ_SILU if silu else 0)
    _written(out)
    return y, out


def _state_out(what, state, out):
    """Where a step writes its state: `out`, or `state` itself; other memory must not overlap it."""
    if not state.is_contiguous():
        raise ValueError(f'{what}: state must be contiguous')
    if out is None:
        return state
    if out.shape != state.shape or out.dtype != state.dtype or out.device != state.device or not out.is_contiguous():
        raise ValueError(f'{what}: state_out must be contiguous and have the shape, type and device of state')
    a, b, n = state.data_ptr(), out.data_ptr(), state.numel() * state.element_size()
    if a != b and a < b + n and b < a + n:
        raise ValueError(f'{what}: state_out overlaps state without being it')
    return out


def _scan_call(x, dt, A, B, C, D, z, bias, h0, seq_off, ld, rows, S, G, flags):
    """The operands as the library takes them; ld: the row distances of x, dt, B, C and z."""
    width, N = A.shape
    return _lib.Scan(x.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z), *ld, A.data_ptr(), _ptr(D), _ptr(bias), _ptr(h0),
                     _ptr(seq_off), rows, S, width, G, N, _DTYPES[x.dtype], flags)


def _scan_rows(x, dt, B, C, z, width, gn):
    """The activation operands as rows, and their distances."""
    x, ldx = _rows(x, width)
    dt, lddt = _rows(dt, width)
    B, ldb = _rows(B, gn)
    C, ldc = _rows(C, gn)
    z, ldz = (None, 0) if z is None else _rows(z, width)
    return x, dt, B, C, z, (ldx, lddt, ldb, ldc, ldz)


def _scan_forward(x, dt, A, B, C, D, z, bias, h0, seq_off, flags, rows, S, G, want_state, keep):
    L = _lib.lib()
    (width, N), dev = A.shape, x.device
    x2, dt2, B2, C2, z2, ld = _scan_rows(x, dt, B, C, z, width, G * N)
    a = _scan_call(x2, dt2, A, B2, C2, D, z2, bias, h0, seq_off, ld, rows, S, G, flags)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    last = torch.empty(S, width, N, dtype=torch.float32, device=dev) if want_state else None
    kept = torch.empty(L.psvae_selective_scan_saved_bytes(rows, S, width, G, N), dtype=torch.uint8, device=dev) if keep else None
    nbytes = L.psvae_selective_scan_scratch_bytes(rows, S, width, G, N, 0)
    sc = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _run('psvae_selective_scan_forward', dev, L.psvae_selective_scan_forward, a, y.data_ptr(), width, _ptr(last), _ptr(kept), _ptr(sc), nbytes)
    return y, last, kept, (x2, dt2, B2, C2, z2, ld)


class SelectiveScanFn(torch.autograd.Function):
    """h[t] = exp(delta A) h[t-1] + delta x B, y = (C h + D x) silu(z) along every sequence; returns (y, last h or None)."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, bias, h0, seq_off, flags, rows, S, G, want_state):
        y, last, kept, (x2, dt2, B2, C2, z2, ld) = _scan_forward(x, dt, A, B, C, D, z, bias, h0, seq_off, flags, rows, S, G, want_state, True)
        ctx.save_for_backward(x2, dt2, A, B2, C2, D, z2, bias, seq_off, kept)
        ctx.call = ld, flags, rows, S, G, x.shape, B.shape
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @_once
    def backward(ctx, dy, dlast):
        L, empty, f32 = _lib.lib(), torch.empty, torch.float32
        x, dt, A, B, C, D, z, bias, seq_off, kept = ctx.saved_tensors
        ld, flags, rows, S, G, shape, bc_shape = ctx.call
        (width, N), dev, dtype = A.shape, A.device, x.dtype
        if dy is None:
            dy = torch.zeros(shape, dtype=dtype, device=dev)
        dy2, lddy = _rows(dy, width)
        if dlast is not None:
            dlast = _f32c(dlast)
        a = _scan_call(x, dt, A, B, C, D, z, bias, None, seq_off, ld, rows, S, G, flags)
        dx, ddt = empty(shape, dtype=dtype, device=dev), empty(shape, dtype=dtype, device=dev)
        dB, dC = empty(bc_shape, dtype=dtype, device=dev), empty(bc_shape, dtype=dtype, device=dev)
        dz = None if z is None else empty(shape, dtype=dtype, device=dev)
        dA = empty(width, N, dtype=f32, device=dev)
        dD = None if D is None else empty(width, dtype=f32, device=dev)
        dbias = None if bias is None else empty(width, dtype=f32, device=dev)
        dh0 = empty(S, width, N, dtype=f32, device=dev) if ctx.needs_input_grad[8] else None
        g = _lib.ScanGrads(dx.data_ptr(), ddt.data_ptr(), dB.data_ptr(), dC.data_ptr(), _ptr(dz), dA.data_ptr(), _ptr(dD), _ptr(dbias), _ptr(dh0))
        nbytes = L.psvae_selective_scan_scratch_bytes(rows, S, width, G, N, 1)
        sc = empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
        _run('psvae_selective_scan_backward', dev, L.psvae_selective_scan_backward, a, kept.data_ptr(), dy2.data_ptr(), lddy, _ptr(dlast), g,
             sc.data_ptr(), nbytes)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dh0, None, None, None, None, None, None


def _scan_operands(what, x, dt, A, B, C, D, z, dt_bias, h0, S):
    """Checks; returns (A, D, dt_bias, h0) in fp32 and the number of groups."""
    width = x.shape[-1]
    if A.dim() != 2 or A.shape[0] != width or not 1 <= A.shape[1] <= 64:
        raise ValueError(f'{what}: A has shape {tuple(A.shape)}, expected [{width}, states] with 1 to 64 states')
    N, lead = A.shape[1], x.shape[:-1]
    G = 1 if B.dim() == x.dim() else B.shape[-2] if B.dim() == x.dim() + 1 else 0
    if G < 1 or width % G:
        raise ValueError(f'{what}: B has shape {tuple(B.shape)}: [.., states] or [.., groups, states] with groups that divide {width}')
    _act(what, 'dt', dt, x, x.shape)
    _act(what, 'B', B, x, (*lead, N) if B.dim() == x.dim() else (*lead, G, N))
    _act(what, 'C', C, x, B.shape)
    if z is not None:
        _act(what, 'z', z, x, x.shape)
    return (_par(what, 'A', A, x, (width, N)), _par(what, 'D', D, x, (width,)), _par(what, 'dt_bias', dt_bias, x, (width,)),
            _par(what, 'h0', h0, x, (S, width, N)), G)


def selective_scan(x, dt, A, B, C, *, D=None, z=None, dt_bias=None, softplus=True, h0=None, seq_off=None, return_state=False):
    """Selective state space scan along every sequence:

        delta = softplus(dt + dt_bias)                                      (softplus=False: dt + dt_bias)
        h[t, d, n] = exp(delta[t, d] A[d, n]) h[t-1, d, n] + delta[t, d] x[t, d] B[t, g, n]
        y[t, d] = (sum_n C[t, g, n] h[t, d, n] + D[d] x[t, d]) * silu(z[t, d])

    x, dt, z [.., width]; B, C [.., N] or [.., G, N], each group shared by width / G neighbouring channels; A [width, N]
    with up to 64 states; D, dt_bias [width]; h0 [S, width, N], the state in front of every sequence (zeros without
    it).  Returns y, with `return_state` (y, the state behind every sequence's end), which carries gradients."""
    what = 'selective_scan'
    _first(what, x, 2, 3)
    rows, S = _sequences(what, x, seq_off)
    A, D, dt_bias, h0, G = _scan_operands(what, x, dt, A, B, C, D, z, dt_bias, h0, S)
    _no_tangent(what, x, dt, A, B, C, D, z, dt_bias, h0)
    flags = (_lib.SEQ_SOFTPLUS if softplus else 0) | (_lib.SEQ_ZERO_OUTSIDE if seq_off is not None else 0)
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, h0):
        y, last = SelectiveScanFn.apply(x, dt, A, B, C, D, z, dt_bias, h0, seq_off, flags, rows, S, G, bool(return_state))
    else:
        y, last = _scan_forward(x, dt, A, B, C, D, z, dt_bias, h0, seq_off, flags, rows, S, G, return_state, False)[:2]
    return (y, last) if return_state else y


def selective_scan_step(x, dt, A, B, C, state, *, D=None, z=None, dt_bias=None, softplus=True, state_out=None):
    """One row of the scan for each of S sequences: x, dt, z [S, width], B, C [S, N] or [S, G, N].  `state` [S, width, N]
    fp32 is moved on, in place or into `state_out`; returns (y, the new state).  No gradients."""
    what = 'selective_scan_step'
    _first(what, x, 2, 2)
    S, width = x.shape
    if state.dtype != torch.float32:
        raise ValueError(f'{what}: state is {state.dtype}, expected torch.float32')
    _no_tangent(what, x, dt, A, B, C, state, D, z, dt_bias, state_out)
    if _wants_grad(x, dt, A, B, C, state, D, z, dt_bias, state_out):
        raise RuntimeError(f'{what} has no backward pass: call it under torch.no_grad() or on detached tensors')
    out = _state_out(what, state, state_out)
    A, D, dt_bias, state, G = _scan_operands(what, x, dt, A, B, C, D, z, dt_bias, state, S)
    x2, dt2, B2, C2, z2, ld = _scan_rows(x, dt, B, C, z, width, G * A.shape[1])
    a = _scan_call(x2, dt2, A, B2, C2, D, z2, dt_bias, state, None, ld, S, S, G, _lib.SEQ_SOFTPLUS if softplus else 0)
    y = torch.empty(S, width, dtype=x.dtype, device=x.device)
    _run('psvae_selective_scan_step', x.device, _lib.lib().psvae_selective_scan_step, a, y.data_ptr(), width, out.data_ptr())
    _written(out)
    return y, out
