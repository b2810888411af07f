// Layer norm over the last dimension, forward and backward, fp32 / bf16 / fp16 rows with fp32 parameters.
//
//   mean = sum x / H,  rstd = 1 / sqrt(sum (x - mean)^2 / H + eps),  xh = (x - mean) rstd,  y = xh w + b
//   g = dy w;  dx = rstd (g - sum g / H - xh sum(g xh) / H);  dw = sum over rows dy xh;  db = sum over rows dy
//
// Both passes are bound by HBM: forward moves x and y once, backward x, dy and dx once.  A row stays in the registers of
// one wave (up to 256 vectors of 16 bytes) or of one workgroup (up to 2048 forward, 1024 backward), so the variance is
// the second pass over registers of the two-pass formula (exact for rows whose mean is large against their spread) at no
// further traffic.  Wider rows are read again for every pass (from L2).  Measured at 32768 x 2048 bf16: forward 57 us
// (4.7 TB/s), backward 86 us (4.7 TB/s; 108 us before it loaded a row ahead) and 4 us for the parameters' sums; a copy
// reaches 5.0 TB/s.  At 3277 x 300 fp32 the three kernels take 5, 7 and 4 us, which the host's time to queue them hides.
#include "seq_device.h"

namespace {

// Sum of one value over the lanes that share a row: a wave, or the four waves of a workgroup.
template <int WPR> __device__ __forceinline__ float row_sum(float v, float* red) {
    v = wave_add(v);
    if constexpr (WPR == 1) return v;
    __syncthreads();                                   // the previous sum's readers are done with `red`
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class T, int V, int WPR, int IT>
__global__ __launch_bounds__(256) void norm_fwd_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                                                       const float* __restrict__ b, T* __restrict__ y, int64_t ldy,
                                                       float* __restrict__ mean, float* __restrict__ rstd, int rows, int H, float eps) {
    __shared__ float red[4];
    const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= rows) return;                           // whole waves (WPR 1) or never (WPR 4)
    const T* xr = x + row * ldx;
    float v[IT][V], s = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * 64 * WPR + lane) * V;
        if (c < H) load_vec<V>(xr + c, v[i]);
        else
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) s += v[i][k];
    }
    const float mu = row_sum<WPR>(s, red) / (float)H;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * 64 * WPR + lane) * V;
        if (c < H)
#pragma unroll
            for (int k = 0; k < V; ++k) { const float d = v[i][k] - mu; s = fmaf(d, d, s); }
    }
    const float rs = 1.f / sqrtf(row_sum<WPR>(s, red) / (float)H + eps);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * 64 * WPR + lane) * V;
        if (c >= H) continue;
        float wv[V], bv[V], o[V];
        if (w) load_vec<V>(w + c, wv);
        if (b) load_vec<V>(b + c, bv);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            o[k] = (v[i][k] - mu) * rs;
            if (w) o[k] *= wv[k];
            if (b) o[k] += bv[k];
        }
        store_vec<V>(y + row * ldy + c, o);
    }
    if (lane == 0) {
        if (mean) mean[row] = mu;
        if (rstd) rstd[row] = rs;
    }
}

// Rows that no workgroup holds in registers: one workgroup a row, three passes over it.
template <class T, int V>
__global__ __launch_bounds__(256) void norm_fwd_wide_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                                                            const float* __restrict__ b, T* __restrict__ y, int64_t ldy,
                                                            float* __restrict__ mean, float* __restrict__ rstd, int H, float eps) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    float s = 0.f;
    for (int c = threadIdx.x * V; c < H; c += 256 * V) {
        float v[V];
        load_vec<V>(xr + c, v);
#pragma unroll
        for (int k = 0; k < V; ++k) s += v[k];
    }
    const float mu = row_sum<4>(s, red) / (float)H;
    s = 0.f;
    for (int c = threadIdx.x * V; c < H; c += 256 * V) {
        float v[V];
        load_vec<V>(xr + c, v);
#pragma unroll
        for (int k = 0; k < V; ++k) { const float d = v[k] - mu; s = fmaf(d, d, s); }
    }
    const float rs = 1.f / sqrtf(row_sum<4>(s, red) / (float)H + eps);
    for (int c = threadIdx.x * V; c < H; c += 256 * V) {
        float v[V], wv[V], bv[V];
        load_vec<V>(xr + c, v);
        if (w) load_vec<V>(w + c, wv);
        if (b) load_vec<V>(b + c, bv);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            v[k] = (v[k] - mu) * rs;
            if (w) v[k] *= wv[k];
            if (b) v[k] += bv[k];
        }
        store_vec<V>(y + row * ldy + c, v);
    }
    if (threadIdx.x == 0) {
        if (mean) mean[row] = mu;
        if (rstd) rstd[row] = rs;
    }
}

// dx, and this workgroup's part of dw and db.  A workgroup takes rows blockIdx.x * ROWS + (0 .. ROWS-1) and on in steps of
// the grid, keeps its columns' sums in registers, joins its waves through LDS and writes them 2 H floats further for every
// workgroup: the parameter gradients cost one pass of 2 H floats per workgroup and no atomics (the order of every sum is
// fixed).  A single workgroup writes the gradients themselves.
template <class T, int V, int WPR, int IT>
__global__ __launch_bounds__(256) void norm_bwd_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                       const float* __restrict__ w, const float* __restrict__ mean,
                                                       const float* __restrict__ rstd, T* __restrict__ dx, int64_t lddx,
                                                       float* __restrict__ dw_out, float* __restrict__ db_out, int rows, int H) {
    extern __shared__ float join[];                    // 2 H floats (WPR 1) or 8 (WPR 4)
    constexpr int ROWS = WPR == 1 ? 4 : 1;
    const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
    float wv[IT][V], dw[IT][V], db[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * 64 * WPR + lane) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) { wv[i][k] = 1.f; dw[i][k] = 0.f; db[i][k] = 0.f; }
        if (w && c < H) load_vec<V>(w + c, wv[i]);
    }
    const float inv = 1.f / (float)H;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    Raw<T, V> gn[IT], xn[IT];                          // the next row, on its way while this one is worked on
    float mun = 0.f, rsn = 0.f;
    auto fetch = [&](int64_t row) {
        mun = mean[row];
        rsn = rstd[row];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * 64 * WPR + lane) * V;
            if (c < H) {
                gn[i].load(dy + row * lddy + c);
                xn[i].load(x + row * ldx + c);
            }
        }
    };
    int64_t row = (int64_t)blockIdx.x * ROWS + (WPR == 1 ? wave : 0);
    if (row < rows) fetch(row);
    for (; row < rows; row += step) {
        const float mu = mun, rs = rsn;
        float g[IT][V], xh[IT][V], s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) { g[i][k] = gn[i][k]; xh[i][k] = xn[i][k]; }
        if (row + step < rows) fetch(row + step);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * 64 * WPR + lane) * V;
            if (c < H) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    xh[i][k] = (xh[i][k] - mu) * rs;
                    db[i][k] += g[i][k];
                    dw[i][k] = fmaf(g[i][k], xh[i][k], dw[i][k]);
                    g[i][k] *= wv[i][k];
                    s0 += g[i][k];
                    s1 = fmaf(g[i][k], xh[i][k], s1);
                }
            }
        }
        if (!dx) continue;
        s0 = wave_add(s0);
        s1 = wave_add(s1);
        if constexpr (WPR == 4) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) { join[wave] = s0; join[4 + wave] = s1; }
            __syncthreads();
            s0 = (join[0] + join[1]) + (join[2] + join[3]);
            s1 = (join[4] + join[5]) + (join[6] + join[7]);
        }
        s0 *= inv;
        s1 *= inv;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * 64 * WPR + lane) * V;
            if (c >= H) continue;
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = rs * (g[i][k] - s0 - xh[i][k] * s1);
            store_vec<V>(dx + row * lddx + c, o);
        }
    }
    if (!dw_out && !db_out) return;
    const int64_t part = (int64_t)blockIdx.x * 2 * H;
    if constexpr (WPR == 1) {
        for (int turn = 0; turn < 4; ++turn) {
            if (wave == turn) {
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    const int c = (i * 64 + lane) * V;
                    if (c >= H) continue;
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        join[c + k] = turn ? join[c + k] + dw[i][k] : dw[i][k];
                        join[H + c + k] = turn ? join[H + c + k] + db[i][k] : db[i][k];
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < H; c += 256) {
            if (dw_out) dw_out[part + c] = join[c];
            if (db_out) db_out[part + c] = join[H + c];
        }
    } else {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * 256 + lane) * V;
            if (c >= H) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if (dw_out) dw_out[part + c + k] = dw[i][k];
                if (db_out) db_out[part + c + k] = db[i][k];
            }
        }
    }
}

// Wide rows: dx from two passes over the row, the parameter gradients from a pass of their own over columns.
template <class T, int V>
__global__ __launch_bounds__(256) void norm_bwd_wide_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                            const float* __restrict__ w, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, T* __restrict__ dx, int64_t lddx, int H) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    const float mu = mean[row], rs = rstd[row];
    float s0 = 0.f, s1 = 0.f;
    for (int c = threadIdx.x * V; c < H; c += 256 * V) {
        float g[V], v[V], wv[V];
        load_vec<V>(dy + row * lddy + c, g);
        load_vec<V>(x + row * ldx + c, v);
        if (w) load_vec<V>(w + c, wv);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (w) g[k] *= wv[k];
            s0 += g[k];
            s1 = fmaf(g[k], (v[k] - mu) * rs, s1);
        }
    }
    s0 = row_sum<4>(s0, red) / (float)H;
    s1 = row_sum<4>(s1, red) / (float)H;
    for (int c = threadIdx.x * V; c < H; c += 256 * V) {
        float g[V], v[V], wv[V];
        load_vec<V>(dy + row * lddy + c, g);
        load_vec<V>(x + row * ldx + c, v);
        if (w) load_vec<V>(w + c, wv);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = rs * ((w ? g[k] * wv[k] : g[k]) - s0 - (v[k] - mu) * rs * s1);
        store_vec<V>(dx + row * lddx + c, v);
    }
}
template <class T, int V>
__global__ __launch_bounds__(256) void norm_param_grad_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              float* __restrict__ partial, int rows, int H) {
    const int c = (blockIdx.y * 256 + threadIdx.x) * V;
    if (c >= H) return;
    float dw[V], db[V];
#pragma unroll
    for (int k = 0; k < V; ++k) dw[k] = db[k] = 0.f;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        float g[V], v[V];
        load_vec<V>(dy + row * lddy + c, g);
        load_vec<V>(x + row * ldx + c, v);
        const float mu = mean[row], rs = rstd[row];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            db[k] += g[k];
            dw[k] = fmaf(g[k], (v[k] - mu) * rs, dw[k]);
        }
    }
    float* out = partial + (int64_t)blockIdx.x * 2 * H + c;
#pragma unroll
    for (int k = 0; k < V; ++k) { out[k] = dw[k]; out[H + k] = db[k]; }
}

// Partial column sums: 16 columns x 16 parts at a time, so that a few hundred columns still fill some CUs.
__global__ __launch_bounds__(256) void column_sums_kernel(const float* __restrict__ partial, int parts, int columns, int width,
                                                          int taps, float* __restrict__ out0, float* __restrict__ out1) {
    __shared__ float red[16][17];
    const int cx = threadIdx.x & 15, px = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + cx;
    float s = 0.f;
    if (c < columns)
#pragma unroll 8
        for (int p = px; p < parts; p += 16) s += partial[(int64_t)p * columns + c];
    red[px][cx] = s;
    __syncthreads();
    if (px == 0 && c < columns) {
        s = 0.f;
#pragma unroll
        for (int p = 0; p < 16; ++p) s += red[p][cx];
        const int k = c / width, d = c - k * width;
        if (k < taps) {
            if (out0) out0[(int64_t)d * taps + k] = s;
        } else if (out1) {
            out1[d] = s;
        }
    }
}

constexpr int NORM_PARTS = 512;   // workgroups of the backward pass: two for every CU

int norm_parts(int64_t rows) {
    // one workgroup for a few rows (no second launch to join the parts); else eight rows to a workgroup before another one
    // is added: the partial sums are 2 H floats each
    const int64_t want = rows <= 16 ? 1 : (rows + 7) / 8;
    return (int)(want < 1 ? 1 : (want > NORM_PARTS ? NORM_PARTS : want));
}

template <class T, int V> int norm_fwd(hipStream_t s, const T* x, int64_t ldx, const float* w, const float* b, T* y, int64_t ldy,
                                       float* mean, float* rstd, int rows, int H, float eps) {
    const int nvec = H / V;
#define PSVAE_NORM_FWD(WPR, IT)                                                                                              \
    hipLaunchKernelGGL((norm_fwd_kernel<T, V, WPR, IT>), dim3(WPR == 1 ? (rows + 3) / 4 : rows), dim3(256), 0, s, x, ldx, w, b, \
                       y, ldy, mean, rstd, rows, H, eps)
    if (nvec <= 64) PSVAE_NORM_FWD(1, 1);
    else if (nvec <= 128) PSVAE_NORM_FWD(1, 2);
    else if (nvec <= 256) PSVAE_NORM_FWD(1, 4);
    else if (nvec <= 512) PSVAE_NORM_FWD(4, 2);
    else if (nvec <= 1024) PSVAE_NORM_FWD(4, 4);
    else if (nvec <= 2048) PSVAE_NORM_FWD(4, 8);
    else hipLaunchKernelGGL((norm_fwd_wide_kernel<T, V>), dim3(rows), dim3(256), 0, s, x, ldx, w, b, y, ldy, mean, rstd, H, eps);
#undef PSVAE_NORM_FWD
    PSVAE_LAUNCH_CHECK();
    return 0;
}

template <class T, int V> int norm_bwd(hipStream_t s, const T* dy, int64_t lddy, const T* x, int64_t ldx, const float* w,
                                       const float* mean, const float* rstd, T* dx, int64_t lddx, float* dw, float* db, int rows,
                                       int H, float* partial) {
    const int nvec = H / V;
    const int parts = norm_parts(rows);
    float* part = dw || db ? partial : nullptr;
    const bool one = parts == 1;
    float *dw_to = one ? dw : part, *db_to = one ? db : (part ? part + H : nullptr);
#define PSVAE_NORM_BWD(WPR, IT)                                                                                            \
    hipLaunchKernelGGL((norm_bwd_kernel<T, V, WPR, IT>), dim3(parts), dim3(256), (WPR == 1 ? 2 * H : 8) * sizeof(float), s, dy, \
                       lddy, x, ldx, w, mean, rstd, dx, lddx, dw_to, db_to, rows, H)
    if (nvec <= 64) PSVAE_NORM_BWD(1, 1);
    else if (nvec <= 128) PSVAE_NORM_BWD(1, 2);
    else if (nvec <= 256) PSVAE_NORM_BWD(1, 4);
    else if (nvec <= 512) PSVAE_NORM_BWD(4, 2);
    else if (nvec <= 1024) PSVAE_NORM_BWD(4, 4);
    else {
        for (int64_t r = 0; dx && r < rows; r += MOST_BLOCKS)
            hipLaunchKernelGGL((norm_bwd_wide_kernel<T, V>), dim3((unsigned)(rows - r < MOST_BLOCKS ? rows - r : MOST_BLOCKS)), dim3(256), 0, s,
                               dy + r * lddy, lddy, x + r * ldx, ldx, w, mean + r, rstd + r, dx + r * lddx, lddx, H);
        if (part) hipLaunchKernelGGL((norm_param_grad_kernel<T, V>), dim3(parts, (nvec + 255) / 256), dim3(256), 0, s, dy, lddy, x, ldx,
                                     mean, rstd, part, rows, H);
    }
#undef PSVAE_NORM_BWD
    PSVAE_LAUNCH_CHECK();
    return part && !(one && nvec <= 1024) ? column_sums(s, part, parts, H, 1, dw, db) : 0;
}

}  // namespace

int column_sums(hipStream_t s, const float* partial, int parts, int width, int taps, float* out0, float* out1) {
    const int columns = width * (taps + 1);
    hipLaunchKernelGGL(column_sums_kernel, dim3((columns + 15) / 16), dim3(256), 0, s, partial, parts, columns, width, taps, out0, out1);
    PSVAE_LAUNCH_CHECK();
    return 0;
}

// Vectors of 16 bytes where every row of every operand starts on one and holds whole ones, single elements otherwise.
static bool norm_vec(int dtype, int H, const void* a, int64_t lda, const void* b, int64_t ldb, const void* c, int64_t ldc,
                     const float* w, const float* bias) {
    const int V = 16 / (int)dtype_bytes(dtype);
    return H % V == 0 && rows_vec(a, lda, V, dtype) && rows_vec(b, ldb, V, dtype) && rows_vec(c, ldc, V, dtype) &&
           rows_vec(w, 0, V, PSVAE_F32) && rows_vec(bias, 0, V, PSVAE_F32);
}

extern "C" int psvae_layer_norm_forward(const void* x, int64_t ldx, const float* weight, const float* bias, void* y, int64_t ldy,
                                        float* mean, float* rstd, int64_t rows, int width, float eps, int dtype, void* stream) {
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > (1 << 23) || ldx < width || ldy < width || !dtype_known(dtype)) return PSVAE_E_SHAPE;
    if (rows == 0) return 0;
    if (!x || !y) return PSVAE_E_NULL;
    const bool vec = norm_vec(dtype, width, x, ldx, y, ldy, nullptr, 0, weight, bias);
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_NORM, 2.0 * rows * width * dtype_bytes(dtype));
    PSVAE_BY_TYPE(dtype, T, {
        constexpr int V = 16 / sizeof(T);
        for (int64_t r = 0; r < rows; r += MOST_BLOCKS) {
            const int n = (int)(rows - r < MOST_BLOCKS ? rows - r : MOST_BLOCKS);
            const T* from = (const T*)x + r * ldx;
            T* to = (T*)y + r * ldy;
            float *const m = mean ? mean + r : nullptr, *const sd = rstd ? rstd + r : nullptr;
            PSVAE_TRY((vec ? norm_fwd<T, V>(s, from, ldx, weight, bias, to, ldy, m, sd, n, width, eps)
                           : norm_fwd<T, 1>(s, from, ldx, weight, bias, to, ldy, m, sd, n, width, eps)));
        }
        return 0;
    });
}

extern "C" size_t psvae_layer_norm_scratch_bytes(int64_t rows, int width) {
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > (1 << 23)) return 0;
    return (size_t)norm_parts(rows) * 2 * width * sizeof(float);
}

extern "C" int psvae_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* weight,
                                         const float* mean, const float* rstd, void* dx, int64_t lddx, float* d_weight,
                                         float* d_bias, int64_t rows, int width, int dtype, void* scratch, size_t scratch_bytes,
                                         void* stream) {
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > (1 << 23) || ldx < width || lddy < width || (dx && lddx < width) || !dtype_known(dtype)) return PSVAE_E_SHAPE;
    if (!dx && !d_weight && !d_bias) return 0;
    if (rows > 0 && (!dy || !x || !mean || !rstd)) return PSVAE_E_NULL;
    if (d_weight || d_bias) {
        if (!scratch) return PSVAE_E_NULL;
        if (!aligned16(scratch)) return PSVAE_E_ALIGN;
        if (scratch_bytes < psvae_layer_norm_scratch_bytes(rows, width)) return PSVAE_E_WORKSPACE;
    } else if (rows == 0) {
        return 0;
    }
    const bool vec = norm_vec(dtype, width, x, ldx, dy, lddy, dx, lddx, weight, nullptr);
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(s, KC_NORM, 3.0 * rows * width * dtype_bytes(dtype));
    PSVAE_BY_TYPE(dtype, T, {
        constexpr int V = 16 / sizeof(T);
        return vec ? norm_bwd<T, V>(s, (const T*)dy, lddy, (const T*)x, ldx, weight, mean, rstd, (T*)dx, lddx, d_weight, d_bias, (int)rows, width, (float*)scratch)
                   : norm_bwd<T, 1>(s, (const T*)dy, lddy, (const T*)x, ldx, weight, mean, rstd, (T*)dx, lddx, d_weight, d_bias, (int)rows, width, (float*)scratch);
    });
}
