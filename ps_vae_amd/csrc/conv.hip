// Short causal convolution along packed sequences, one filter a channel, with its optional SiLU: forward, backward and
// the form for single tokens.
//
//   pre[t, d] = b[d] + sum_k w[d, k] x[t - W + 1 + k, d]      y = silu ? pre / (1 + exp(-pre)) : pre
//   dpre = silu ? dy sig(pre) (1 + pre (1 - sig(pre))) : dy
//   dx[t, d] = sum_k w[d, k] dpre[t + W - 1 - k, d]            dw[d, k] = sum_t dpre[t, d] x[t - W + 1 + k, d]
//
// Rows in front of a sequence come from its `state` (the last W - 1 inputs before it) or are zero; no product crosses a
// sequence border.  All passes are bound by HBM: a lane owns 16 bytes of channels and walks down a stretch of rows with
// the W rows it needs in registers, so every input row is read once per stretch plus W - 1 rows of run-up.
// Stretches are laid over the packed rows and not over the sequences (a lane finds its sequence by bisection and then
// follows the borders), so that one long and a thousand short sequences load the chip alike.  Rows are loaded four at a
// time, one group ahead, and a group without a border goes through without a test.  Measured at 8 x 2048 x 2048 bf16, four
// taps: forward 33 us (4.1 TB/s; 49 us with no group ahead), backward 58 us (3.5 TB/s; 107 us with eight channels a lane and
// two rows at a time) and 4 us for the parameters' sums; a copy reaches 5.0 TB/s.
#include "seq_device.h"

namespace {

// The sequence that row t belongs to: the last one that begins at or before t and is not empty behind t.  Behind the last
// one it is S, which begins so far off that no row counts as one in front of it (it has no state).
struct Walk { int s, begin, end; };
__device__ __forceinline__ Walk walk_to(const int32_t* off, int S, int T, int t) {
    if (!off) {
        const int L = T / S, s = t / L;
        return {s, s * L, s * L + L};
    }
    int lo = 0, hi = S;                                  // first sequence whose end lies behind t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (off[mid + 1] > t) hi = mid; else lo = mid + 1;
    }
    if (lo == S) return {S, INT32_MAX - 16, INT32_MAX - 16};
    const SeqBounds b = seq_bounds(off, lo, S, T);
    return {lo, b.begin, b.end};
}

// Input row `t` of sequence w (t may lie up to W - 1 rows in front of it).
template <class T, int V>
__device__ __forceinline__ void input_row(const T* x, int64_t ldx, const T* state, const Walk& w, int t, int back, int D, int c, float (&v)[V]) {
    if (t >= w.begin) load_vec<V>(x + (int64_t)t * ldx + c, v);
    else if (state && w.begin - t <= back) load_vec<V>(state + ((int64_t)w.s * back + back - (w.begin - t)) * D + c, v);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
}

struct ConvShape { int T, D, S, R, lanes; int flags; };   // R rows a stretch, `lanes` lanes side by side in a row
constexpr int GROUP = 4;   // rows loaded at a time, while the group before them is worked on

template <class T, int V, int W>
__global__ __launch_bounds__(256) void conv_fwd_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                                                       const float* __restrict__ b, T* __restrict__ y, int64_t ldy,
                                                       const int32_t* __restrict__ off, const T* __restrict__ state, ConvShape q) {
    const int c = (blockIdx.y * q.lanes + threadIdx.x % q.lanes) * V;
    const int t0 = (blockIdx.x * (256 / q.lanes) + threadIdx.x / q.lanes) * q.R;
    if (c >= q.D || t0 >= q.T) return;
    const int t1 = min(t0 + q.R, q.T);
    float wv[W][V], bv[V], win[W][V];
    Raw<T, V> now[GROUP], next[GROUP];
    x += c;
    y += c;
    auto fetch = [&](int t) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
            if (t + j < t1) next[j].load(x + (int64_t)(t + j) * ldx);
    };
    fetch(t0);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bv[i] = b ? b[c + i] : 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) wv[k][i] = w[(int64_t)(c + i) * W + k];
    }
    Walk at = walk_to(off, q.S, q.T, t0);
    auto run_up = [&](int t) {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) input_row<T, V>(x - c, ldx, state, at, t - W + 1 + k, W - 1, q.D, c, win[k + 1]);
    };
    auto row = [&](int t, const Raw<T, V>& in) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) win[k][i] = win[k + 1][i];
            win[W - 1][i] = in[i];
            float pre = bv[i];
#pragma unroll
            for (int k = 0; k < W; ++k) pre = fmaf(wv[k][i], win[k][i], pre);
            o[i] = q.flags & PSVAE_SEQ_SILU ? pre * sigmoidf(pre) : pre;
        }
        store_vec<V>(y + (int64_t)t * ldy, o);
    };
    run_up(t0);
    for (int tb = t0; tb < t1; tb += GROUP) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) now[j] = next[j];
        fetch(tb + GROUP);
        if (tb > at.begin && tb + GROUP <= min(at.end, t1)) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j) row(tb + j, now[j]);
            continue;
        }
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {               // a border of a sequence or of the stretch lies in this group
            const int t = tb + j;
            if (t >= t1) break;
            if (t >= at.end && at.s < q.S) at = walk_to(off, q.S, q.T, t);   // the next sequence that has rows, or none
            if (t == at.begin) run_up(t);
            if (at.s < q.S && t >= at.begin) {
                row(t, now[j]);
            } else if (q.flags & PSVAE_SEQ_ZERO_OUTSIDE) {
                float zero[V];
#pragma unroll
                for (int i = 0; i < V; ++i) zero[i] = 0.f;
                store_vec<V>(y + (int64_t)t * ldy, zero);
            }
        }
    }
}

// The last W - 1 inputs of every sequence (with its own state in front where it is shorter).
template <class T>
__global__ __launch_bounds__(256) void conv_state_kernel(const T* __restrict__ x, int64_t ldx, const int32_t* __restrict__ off,
                                                         const T* __restrict__ state, T* __restrict__ out, int S, int T_, int D, int back) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)S * back * D; i += (int64_t)gridDim.x * 256) {
        const int d = (int)(i % D), k = (int)(i / D % back), s = (int)(i / ((int64_t)D * back));
        const SeqBounds q = seq_bounds(off, s, S, T_);
        const int t = q.end - back + k;
        out[i] = t >= q.begin ? x[(int64_t)t * ldx + d]
                              : (state ? state[((int64_t)s * back + back - (q.begin - t)) * D + d] : (T)0.f);
    }
}

// dx, and this workgroup's part of dw and db: partial[blockIdx.x][W + 1][D].  The pre-activation is computed again from
// x (cheaper than keeping it: it would be one more read and one more write of the whole activation).
template <class T, int V, int W>
__global__ __launch_bounds__(256) void conv_bwd_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                       const float* __restrict__ w, const float* __restrict__ b, T* __restrict__ dx,
                                                       int64_t lddx, float* __restrict__ partial, const int32_t* __restrict__ off,
                                                       const T* __restrict__ state, ConvShape q) {
    extern __shared__ float join[];                      // 256 V floats
    const int lane = threadIdx.x % q.lanes, stretch = threadIdx.x / q.lanes, stretches = 256 / q.lanes;
    const int c = (blockIdx.y * q.lanes + lane) * V;
    const int t0 = (blockIdx.x * stretches + stretch) * q.R;
    const int t1 = min(t0 + q.R, q.T);
    float wv[W][V], bv[V], win[W][V], ring[W][V], dw[W][V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bv[i] = db[i] = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) wv[k][i] = win[k][i] = ring[k][i] = dw[k][i] = 0.f;
    }
    if (c < q.D && t0 < q.T) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bv[i] = b ? b[c + i] : 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) wv[k][i] = w[(int64_t)(c + i) * W + k];
        }
        // ring[k]: the gradient gathered so far for row t - W + 1 + k
        auto emit = [&](int row, const float (&g)[V]) {
            if (dx && row >= t0 && row < t1) store_vec<V>(dx + (int64_t)row * lddx + c, g);
        };
        Walk at = walk_to(off, q.S, q.T, t0);
        const int last = min(t1 + W - 1, q.T);          // rows behind the stretch that its own rows' gradients come from, too
        Raw<T, V> xr[GROUP], gr[GROUP], xn[GROUP], gn[GROUP];
        auto fetch = [&](int t) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j)
                if (t + j < last) {
                    xn[j].load(x + (int64_t)(t + j) * ldx + c);
                    gn[j].load(dy + (int64_t)(t + j) * lddy + c);
                }
        };
        auto run_up = [&](int t) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) input_row<T, V>(x, ldx, state, at, t - W + 1 + k, W - 1, q.D, c, win[k + 1]);
        };
        auto row = [&](const Raw<T, V>& xin, const Raw<T, V>& gin, bool own) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int k = 0; k + 1 < W; ++k) win[k][i] = win[k + 1][i];
                win[W - 1][i] = xin[i];
                float g = gin[i];
                if (q.flags & PSVAE_SEQ_SILU) {
                    float pre = bv[i];
#pragma unroll
                    for (int k = 0; k < W; ++k) pre = fmaf(wv[k][i], win[k][i], pre);
                    const float sg = sigmoidf(pre);
                    g *= sg * (1.f + pre * (1.f - sg));
                }
                // shift the ring down by one row, then give every row of the window its product
#pragma unroll
                for (int k = 0; k + 1 < W; ++k) ring[k][i] = fmaf(wv[k][i], g, ring[k + 1][i]);
                ring[W - 1][i] = wv[W - 1][i] * g;
                if (own) {
                    db[i] += g;
#pragma unroll
                    for (int k = 0; k < W; ++k) dw[k][i] = fmaf(g, win[k][i], dw[k][i]);
                }
            }
        };
        fetch(t0);
        run_up(t0);
        bool done = false;
        for (int tb = t0; tb < last && !done; tb += GROUP) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j) { xr[j] = xn[j]; gr[j] = gn[j]; }
            fetch(tb + GROUP);
            if (tb - W + 1 >= max(t0, at.begin) && tb > at.begin && tb + GROUP <= min(at.end, t1)) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    row(xr[j], gr[j], true);
                    if (dx) store_vec<V>(dx + (int64_t)(tb + j - W + 1) * lddx + c, ring[0]);
                }
                continue;
            }
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                const int t = tb + j;
                if (t >= last || done) break;
                if (t >= at.end && at.s < q.S) {
                    // the sequence is over: its last W - 1 rows have all that they get
#pragma unroll
                    for (int k = 1; k < W; ++k)
                        if (t - W + k >= at.begin) emit(t - W + k, ring[k]);
#pragma unroll
                    for (int i = 0; i < V; ++i)
#pragma unroll
                        for (int k = 0; k < W; ++k) ring[k][i] = 0.f;
                    if (t >= t1) { done = true; break; }
                    at = walk_to(off, q.S, q.T, t);
                }
                if (t == at.begin) run_up(t);
                if (at.s >= q.S || t < at.begin) {
                    if (q.flags & PSVAE_SEQ_ZERO_OUTSIDE) {
                        float zero[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) zero[i] = 0.f;
                        emit(t, zero);
                    }
                    continue;
                }
                row(xr[j], gr[j], t < t1);
                if (t - W + 1 >= at.begin) emit(t - W + 1, ring[0]);
            }
        }
        // the walk ended behind the last row: what is still in the ring is complete
        if (!done && last == q.T && at.s < q.S)
#pragma unroll
            for (int k = 1; k < W; ++k)
                if (q.T - W + k >= at.begin && q.T - W + k < at.end) emit(q.T - W + k, ring[k]);
    }
    if (!partial) return;
    // join the stretches of this workgroup, one quantity after the other, in the stretches' order
    float* out = partial + (int64_t)blockIdx.x * (W + 1) * q.D;
#pragma unroll
    for (int k = 0; k <= W; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) join[threadIdx.x * V + i] = k < W ? dw[k < W ? k : 0][i] : db[i];
        __syncthreads();
        for (int e = threadIdx.x; e < q.lanes * V; e += 256) {
            float s = 0.f;
            for (int p = 0; p < stretches; ++p) s += join[p * q.lanes * V + e];
            const int col = blockIdx.y * q.lanes * V + e;
            if (col < q.D) out[(int64_t)k * q.D + col] = s;
        }
    }
}

// One token for each of S sequences.  A lane owns its channels' whole state, so `state_out` may be `state`.
template <class T, int V, int W>
__global__ __launch_bounds__(256) void conv_step_kernel(const T* __restrict__ x, int64_t ldx, const T* state, T* state_out,
                                                        const float* __restrict__ w, const float* __restrict__ b, T* __restrict__ y,
                                                        int64_t ldy, int S, int D, int flags) {
    const int per = D / V;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)S * per; i += (int64_t)gridDim.x * 256) {
        const int64_t s = i / per;
        const int c = (int)(i - s * per) * V;
        float win[W][V], o[V];
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) load_vec<V>(state + (s * (W - 1) + k) * D + c, win[k]);
        load_vec<V>(x + s * ldx + c, win[W - 1]);
#pragma unroll
        for (int i2 = 0; i2 < V; ++i2) {
            float pre = b ? b[c + i2] : 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) pre = fmaf(w[(int64_t)(c + i2) * W + k], win[k][i2], pre);
            o[i2] = flags & PSVAE_SEQ_SILU ? pre * sigmoidf(pre) : pre;
        }
        store_vec<V>(y + s * ldy + c, o);
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) store_vec<V>(state_out + (s * (W - 1) + k) * D + c, win[k + 1]);
    }
}

// Lanes side by side in a row: the smallest power of two that covers the channels, at most a wave (whose access is then
// one run of 1 KB); the other lanes of the workgroup take further stretches.
int conv_lanes(int nvec) {
    int l = 8;
    while (l < 64 && l < nvec) l *= 2;
    return l;
}
// Rows a stretch: long ones read less twice (W - 1 rows of run-up), short ones make more workgroups.  The longest that
// still gives four workgroups to every CU, between 8 and 64.
int conv_rows(int64_t T, int nvec, int lanes) {
    int R = 64;
    while (R > 8 && (T + R * (256 / lanes) - 1) / (R * (256 / lanes)) * ((nvec + lanes - 1) / lanes) < 1024) R /= 2;
    return R;
}
// Channels of a lane where rows allow vectors: 16 bytes forward; four backward and for more than four taps, whose windows,
// filters and sums would otherwise leave registers for a single wave of a SIMD.
int conv_vec(int dtype, int W, bool backward) { return dtype == PSVAE_F32 || backward || W > 4 ? 4 : 8; }

unsigned blocks_of(int64_t n) { return (unsigned)((n + 255) / 256 < MOST_BLOCKS ? (n + 255) / 256 : MOST_BLOCKS); }

struct ConvPlan { ConvShape q; int V, gx, gy; };
ConvPlan conv_plan(int64_t T, int D, int S, int V, int flags) {
    const int nvec = (D + V - 1) / V, lanes = conv_lanes(nvec), R = conv_rows(T, nvec, lanes);
    const int per = R * (256 / lanes);
    return {{(int)T, D, S, R, lanes, flags}, V, (int)((T + per - 1) / per), (nvec + lanes - 1) / lanes};
}

template <class T, int V, int W> struct ConvRun {
    static int fwd(hipStream_t s, const ConvPlan& p, const void* x, int64_t ldx, const float* w, const float* b, void* y, int64_t ldy,
                   const int32_t* off, const void* state) {
        hipLaunchKernelGGL((conv_fwd_kernel<T, V, W>), dim3(p.gx, p.gy), dim3(256), 0, s, (const T*)x, ldx, w, b, (T*)y, ldy, off,
                           (const T*)state, p.q);
        PSVAE_LAUNCH_CHECK();
        return 0;
    }
    static int step(hipStream_t s, const void* x, int64_t ldx, const void* state, void* state_out, const float* w, const float* b, void* y,
                    int64_t ldy, int S, int D, int flags) {
        const int64_t n = (int64_t)S * (D / V);
        hipLaunchKernelGGL((conv_step_kernel<T, V, W>), dim3(blocks_of(n)), dim3(256), 0, s, (const T*)x, ldx, (const T*)state,
                           (T*)state_out, w, b, (T*)y, ldy, S, D, flags);
        PSVAE_LAUNCH_CHECK();
        return 0;
    }
    static int bwd(hipStream_t s, const ConvPlan& p, const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* w,
                   const float* b, void* dx, int64_t lddx, float* partial, const int32_t* off, const void* state) {
        hipLaunchKernelGGL((conv_bwd_kernel<T, V, W>), dim3(p.gx, p.gy), dim3(256), partial ? 256 * V * sizeof(float) : 0, s, (const T*)dy,
                           lddy, (const T*)x, ldx, w, b, (T*)dx, lddx, partial, off, (const T*)state, p.q);
        PSVAE_LAUNCH_CHECK();
        return 0;
    }
};

// Calls `call` of the ConvRun for (type, vector width V, taps).
#define PSVAE_CONV_TAPS(T, V, W, call)                 \
    switch (W) {                                       \
        case 1: return ConvRun<T, V, 1>::call;         \
        case 2: return ConvRun<T, V, 2>::call;         \
        case 3: return ConvRun<T, V, 3>::call;         \
        case 4: return ConvRun<T, V, 4>::call;         \
        case 5: return ConvRun<T, min4(V), 5>::call;   \
        case 6: return ConvRun<T, min4(V), 6>::call;   \
        case 7: return ConvRun<T, min4(V), 7>::call;   \
        default: return ConvRun<T, min4(V), 8>::call;  \
    }
#define PSVAE_CONV_RUN(dtype, V, W, call)                                    \
    PSVAE_BY_TYPE(dtype, T, {                                                \
        if ((V) == 1) { PSVAE_CONV_TAPS(T, 1, W, call) }                     \
        else { PSVAE_CONV_TAPS(T, (int)(16 / sizeof(T)), W, call) }          \
    })
#define PSVAE_CONV_RUN4(dtype, V, W, call)                                   \
    PSVAE_BY_TYPE(dtype, T, {                                                \
        if ((V) == 1) { PSVAE_CONV_TAPS(T, 1, W, call) }                     \
        else { PSVAE_CONV_TAPS(T, 4, W, call) }                              \
    })
constexpr int min4(int v) { return v < 4 ? v : 4; }

bool conv_sizes_ok(int64_t T, int S, int D, int W, int dtype, const void* off) {
    if (T < 0 || T > INT32_MAX - 64 * 64 || S < 0 || D < 1 || D > (1 << 21) || W < 1 || W > 8 || !dtype_known(dtype)) return false;
    return off || S == 0 ? (S > 0 || T == 0) : T % S == 0;
}

}  // namespace

extern "C" int psvae_causal_conv_forward(const void* x, int64_t ldx, const float* weight, const float* bias, void* y, int64_t ldy,
                                         const int32_t* seq_off, const void* state, void* state_out, int64_t T, int S, int D, int W,
                                         int dtype, int flags, void* stream) {
    if (!conv_sizes_ok(T, S, D, W, dtype, seq_off) || ldx < D || ldy < D || (flags & ~(PSVAE_SEQ_SILU | PSVAE_SEQ_ZERO_OUTSIDE))) return PSVAE_E_SHAPE;
    if (!weight || (T > 0 && (!x || !y))) return PSVAE_E_NULL;
    if (state_out && state_out == state) return PSVAE_E_SHAPE;
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SEQ_CONV, 2.0 * T * D * dtype_bytes(dtype));
    if (state_out && S > 0 && W > 1) {
        const int64_t n = (int64_t)S * (W - 1) * D;
        PSVAE_BY_TYPE(dtype, E, {
            hipLaunchKernelGGL((conv_state_kernel<E>), dim3(blocks_of(n)), dim3(256), 0, s, (const E*)x, ldx, seq_off,
                               (const E*)state, (E*)state_out, S, (int)T, D, W - 1);
        });
        PSVAE_LAUNCH_CHECK();
    }
    if (T == 0) return 0;
    const int V = conv_vec(dtype, W, false);
    const bool vec = D % V == 0 && rows_vec(x, ldx, V, dtype) && rows_vec(y, ldy, V, dtype) && rows_vec(state, D, V, dtype);
    const ConvPlan p = conv_plan(T, D, S, vec ? V : 1, flags);
    PSVAE_CONV_RUN(dtype, p.V, W, fwd(s, p, x, ldx, weight, bias, y, ldy, seq_off, state));
}

extern "C" size_t psvae_causal_conv_scratch_bytes(int64_t T, int D, int W, int dtype) {
    if (!conv_sizes_ok(T, 1, D, W, dtype, nullptr)) return 0;
    const ConvPlan a = conv_plan(T, D, 1, 4, 0), b = conv_plan(T, D, 1, 1, 0);   // either may be taken
    return (size_t)((a.gx > b.gx ? a.gx : b.gx) + 1) * (W + 1) * D * sizeof(float);
}

extern "C" int psvae_causal_conv_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* weight,
                                          const float* bias, void* dx, int64_t lddx, float* d_weight, float* d_bias,
                                          const int32_t* seq_off, const void* state, int64_t T, int S, int D, int W, int dtype,
                                          int flags, void* scratch, size_t scratch_bytes, void* stream) {
    if (!conv_sizes_ok(T, S, D, W, dtype, seq_off) || ldx < D || lddy < D || (dx && lddx < D) || (flags & ~(PSVAE_SEQ_SILU | PSVAE_SEQ_ZERO_OUTSIDE))) return PSVAE_E_SHAPE;
    if (!weight || (T > 0 && (!dy || !x))) return PSVAE_E_NULL;
    const bool params = d_weight || d_bias;
    if (!dx && !params) return 0;
    if (params) {
        if (!scratch) return PSVAE_E_NULL;
        if (!aligned16(scratch)) return PSVAE_E_ALIGN;
        if (scratch_bytes < psvae_causal_conv_scratch_bytes(T, D, W, dtype)) return PSVAE_E_WORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SEQ_CONV, 3.0 * T * D * dtype_bytes(dtype));
    float* partial = params ? (float*)scratch : nullptr;
    int parts = 0;
    if (T > 0) {
        const int V = conv_vec(dtype, W, true);
        const bool vec = D % V == 0 && rows_vec(x, ldx, V, dtype) && rows_vec(dy, lddy, V, dtype) && rows_vec(dx, lddx, V, dtype) &&
                         rows_vec(state, D, V, dtype);
        const ConvPlan p = conv_plan(T, D, S, vec ? V : 1, flags);
        parts = p.gx;
        const int rc = [&]() -> int {
            PSVAE_CONV_RUN4(dtype, p.V, W, bwd(s, p, dy, lddy, x, ldx, weight, bias, dx, lddx, partial, seq_off, state));
        }();
        PSVAE_TRY(rc);
    }
    return params ? column_sums(s, partial, parts, D, W, d_weight, d_bias) : 0;
}

extern "C" int psvae_causal_conv_step(const void* x, int64_t ldx, const void* state, void* state_out, const float* weight,
                                      const float* bias, void* y, int64_t ldy, int S, int D, int W, int dtype, int flags, void* stream) {
    if (S < 0 || D < 1 || D > (1 << 21) || W < 1 || W > 8 || !dtype_known(dtype) || ldx < D || ldy < D || (flags & ~PSVAE_SEQ_SILU)) return PSVAE_E_SHAPE;
    if (S == 0) return 0;
    if (!x || !weight || !y || (W > 1 && (!state || !state_out))) return PSVAE_E_NULL;
    const int V = conv_vec(dtype, W, false);
    const bool vec = D % V == 0 && rows_vec(x, ldx, V, dtype) && rows_vec(y, ldy, V, dtype) && rows_vec(state, D, V, dtype) && rows_vec(state_out, D, V, dtype);
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_SEQ_CONV, 2.0 * S * D * W * dtype_bytes(dtype));
    PSVAE_CONV_RUN(dtype, vec ? V : 1, W, step(s, x, ldx, state, state_out, weight, bias, y, ldy, S, D, flags));
}
